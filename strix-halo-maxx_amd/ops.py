"""Drop-in op classes over the C-ABI HIP kernels.

They keep the reference's operator protocol so the per-model forwards read like the reference's:
  * Linear:   cls(weight, bias, dtype); __call__(x, gelu=False, res=None) -> x.shape[:-1] + (N,) bf16; class flags
              fused_gelu / fused_res (moondream/gpu/md2fast.py:33-40, :55-67; hgemm.py:139-178)
  * Attention: Attn(H, T, D); __call__(q, k, v, out=None) with q, k, v (B, H, T, D) views whose last dim is
              contiguous -> (B, T, H*D) (hattn.py:17-37)
Every call launches asynchronously on torch's current stream; nothing here synchronises, so a forward made of these
calls can be captured into a HIP graph.
"""
import json
import os

import torch

from . import _lib
from ._lib import call, ptr, stream

BF = torch.bfloat16
ACT = {None: 0, False: 0, True: 1, "tanh": 1, "erf": 2, "glu": 3}


def _rows(x, K):
    """2-D view (M, K) of x with unit column stride and a 16-byte aligned row stride (copies only if needed)."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(1) != 1 or x2.stride(0) % 8 or x2.data_ptr() % 16:
        x2 = x2.contiguous()
    return x2


class Workspace:
    """Split-K scratch shared by every GEMM on one device: fp32 partial tiles + per-tile arrival counters.

    Grown on demand outside graph capture (call reserve() before capturing); counters start at zero and every
    kernel that uses them leaves them at zero. Kernels on one stream serialise, so one buffer serves all layers (as
    the reference's single split-K workspace, moondream/gpu/hgemm.py:78-83); concurrent GEMMs on two streams would
    race on it. A buffer that was outgrown stays: graphs captured before write to it when they are replayed. (Each is at
    least a quarter larger than the one before, so all of them hold less than five times the last.)
    """
    _by_dev = {}

    def __init__(self, device):
        self.dev = device
        self.ws = torch.empty(0, device=device, dtype=torch.float32)
        self.cnt = torch.zeros(0, device=device, dtype=torch.int32)
        self.outgrown = []

    @classmethod
    def get(cls, device):
        d = torch.device(device)
        key = d.index if d.index is not None else torch.cuda.current_device()
        if key not in cls._by_dev:
            cls._by_dev[key] = cls(d)
        return cls._by_dev[key]

    def reserve(self, elems, counters):
        if elems > self.ws.numel():
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("split-K workspace must be reserved before graph capture")
            self.outgrown.append(self.ws)
            self.ws = torch.empty(int(elems * 1.25) + 1024, device=self.dev, dtype=torch.float32)
        if counters > self.cnt.numel():
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("split-K counters must be reserved before graph capture")
            torch.cuda.synchronize(self.dev)
            self.outgrown.append(self.cnt)
            self.cnt = torch.zeros(int(counters * 1.25) + 64, device=self.dev, dtype=torch.int32)


_TUNED = {}  # (M, N, Kw) -> (cfg, splits), shared by every layer of that shape

# Fixed tile table for MI355X (built by `python -m strix_halo_maxx_amd.tune` from in-context timings: each shape timed
# on the sequence of launches it runs in, with its real cache state). Shapes it lists skip the autotuner, so every
# process runs the same kernels; the reference's pick_cfg has the same two tiers (FIXED table, then timing,
# moondream/gpu/hgemm.py:47-76).
_TABLE_FILE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "gemm_table_gfx950.json")


def _load_table():
    try:
        with open(_TABLE_FILE) as f:
            d = json.load(f)
    except (OSError, ValueError):
        return {}, {}
    conv = lambda m: {tuple(int(v) for v in k.split(",")): tuple(int(v) for v in c) for k, c in m.items()}
    return conv(d.get("fused", {})), conv(d.get("partial", {}))


_FIXED, _FIXED_P = _load_table()


def _ws_need(cfg, splits, M, N):
    lib = _lib.load()
    return lib.mx_gemm_ws_elems(cfg, splits, M, N), lib.mx_gemm_ws_counters(cfg, splits, M, N)


class MxLin:
    """bf16 Linear on the MFMA GEMM: y = epi(x W^T + b) with epi = [GELU tanh|erf] then [+ res], torch's rounding.

    Weights stay in torch's (N, K) layout, zero-padded along K to a multiple of 64 (the kernel's k-step); inputs need
    K columns (K rounded up to 8: the 588-wide patch embedding takes its input zero-padded to 592 by the patchify
    kernel). Bias is held in fp32, as the reference's HLin does (hgemm.py:153). The tile config and split-K factor
    are chosen per (M, N, K) by timing every candidate once (the reference's pick_cfg autotune, hgemm.py:52-76),
    or taken from the library's default pick when tuning is off.
    """
    fused_gelu = True
    fused_res = True
    autotune = True
    use_table = True

    def __init__(self, weight, bias, dtype=BF, device="cuda"):
        assert dtype == BF, "bf16 only"
        w = weight.detach().to(device=device, dtype=BF)
        self.N, self.K0 = w.shape
        self.K = (self.K0 + 7) // 8 * 8          # input columns expected
        self.Kw = (self.K0 + 63) // 64 * 64      # padded weight row
        if self.N % 4:
            raise ValueError(f"N={self.N} must be a multiple of 4")
        if self.Kw == self.K0 and w.stride(1) == 1 and w.stride(0) % 8 == 0 and w.data_ptr() % 16 == 0:
            self.w = w  # already in the kernel's layout: share the storage (e.g. a row slice of a fused weight)
        else:
            wp = torch.zeros(self.N, self.Kw, device=device, dtype=BF)
            wp[:, :self.K0] = w
            self.w = wp
        self.Kp = self.K                         # width of the input this layer reads
        self.b = None if bias is None else bias.detach().to(device=device, dtype=torch.float32).contiguous()
        self.cfgs = {}  # M -> (cfg, splits); absent: tuned (or library pick) on first use
        self.dev = self.w.device

    def _launch(self, cfg, splits, x2, y2, M, a, r2, ldr, r_rows, ws, act_cols=0, act_from=0):
        """splits > 0: mx_gemm_bf16 (in-kernel split-K when > 1); splits = -S: the fence-free split-K, raw partials of
        S splits into the workspace (mx_gemm_bf16_partial) then the epilogue over their sum (mx_gemm_reduce)."""
        lib = _lib.load()
        if splits < 0:
            S, N = -splits, self.N
            if S * M * N > ws.ws.numel():
                return -3
            P = ws.ws[:S * M * N].view(S, M, N)
            rc = _partial(self, cfg, S, x2, P, M)
            if rc != 0:
                return rc
            fn = lib.mx_gemm_reduce_act_from if act_from else lib.mx_gemm_reduce
            return fn(stream(), P.data_ptr(), S, M * N, N, ptr(self.b), ptr(r2), ldr, r_rows, y2.data_ptr(),
                      y2.stride(0), M, N, a, act_from or act_cols)
        fn = lib.mx_gemm_bf16_act_from if act_from else lib.mx_gemm_bf16
        return fn(
            stream(), cfg, splits, x2.data_ptr(), x2.stride(0), self.w.data_ptr(), self.w.stride(0), ptr(self.b),
            ptr(r2), ldr, r_rows, y2.data_ptr(), y2.stride(0), M, self.N, self.K, self.Kw, a, act_from or act_cols,
            ptr(ws.ws), ws.ws.numel(), ptr(ws.cnt), ws.cnt.numel())

    def _pick(self, M, x2, y2, a, r2, ldr, r_rows, ws):
        key = (M, self.N, self.Kw)
        if key in _TUNED:
            return _TUNED[key]
        if MxLin.use_table and key in _FIXED:
            _TUNED[key] = _FIXED[key]
            return _TUNED[key]
        lib = _lib.load()
        if not MxLin.autotune or torch.cuda.is_current_stream_capturing():
            p = lib.mx_gemm_pick(M, self.N, self.Kw)
            c = (p // 16, p % 16)
        else:
            c = tune_gemm(self, M, x2, y2, a, r2, ldr, r_rows, ws)
        _TUNED[key] = c
        return c

    def __call__(self, x, gelu=False, res=None, pre=None, act=None, out=None, act_cols=0, act_from=0):
        """act: None / "tanh" / "erf" / "glu" (gated GELU on interleaved (gate, up) weight rows: output width N / 2);
        act_cols > 0 limits the activation to output columns < act_cols, act_from > 0 to columns >= act_from (a
        multiple of 4; not both, and not with "glu")."""
        if act_from and (act_cols > 0 or act == "glu"):
            raise ValueError("act_from goes with neither act_cols nor glu")
        a = ACT[act if act is not None else gelu]
        Nout = self.N // 2 if a == 3 else self.N
        x2 = _rows(x, self.K)
        if x2.shape[1] == self.K0 and self.K != self.K0:
            xp = torch.zeros(x2.shape[0], self.K, device=x2.device, dtype=BF)
            xp[:, :self.K0] = x2
            x2 = xp
        if x2.shape[1] != self.K:
            raise ValueError(f"input width {x2.shape[1]} != {self.K}")
        M = x2.shape[0]
        y = out if out is not None else torch.empty(M, Nout, device=x2.device, dtype=BF)
        if y.shape[-1] != Nout or y.stride(-1) != 1:
            raise ValueError("out must be (M, N) with unit column stride")
        y2 = y.view(-1, Nout) if y.dim() != 2 else y
        r2, r_rows, ldr = None, 0, 0
        if res is not None:
            r2 = res.reshape(-1, self.N)
            if r2.stride(1) != 1:
                r2 = r2.contiguous()
            ldr = r2.stride(0)
            if r2.shape[0] != M:
                if M % r2.shape[0]:
                    raise ValueError("residual rows must equal or divide the output rows")
                r_rows = r2.shape[0]
        ws = Workspace.get(x2.device)
        cfg, splits = self.cfgs.get(M) or self._pick(M, x2, y2, a, r2, ldr, r_rows, ws)
        if splits > 1:
            ws.reserve(*_ws_need(cfg, splits, M, self.N))
        elif splits < 0:
            ws.reserve(-splits * M * self.N, 0)
        _lib.check(self._launch(cfg, splits, x2, y2, M, a, r2, ldr, r_rows, ws, act_cols, act_from), "mx_gemm_bf16")
        return y2.view(*x.shape[:-1], Nout) if out is None else y

    def partial(self, x, out=None):
        """Raw fp32 split-K partial sums of x W^T, shape (splits, M, N), for a consumer that adds them in order
        together with the bias (residual_layernorm). The tile config and split count are tuned per (M, N, K)."""
        x2 = _rows(x, self.K)
        if x2.shape[1] != self.K:
            raise ValueError(f"input width {x2.shape[1]} != {self.K}")
        M = x2.shape[0]
        cfg, sp = _partial_cfg(self, M, x2)
        P = out if out is not None else torch.empty(sp, M, self.N, device=x2.device, dtype=torch.float32)
        if P.shape != (sp, M, self.N) or P.stride(2) != 1:
            raise ValueError("out must be (splits, M, N) fp32 with unit column stride")
        _lib.check(_partial(self, cfg, sp, x2, P, M), "mx_gemm_bf16_partial")
        return P

    def res_ln(self, x, res, ln, eps=1e-5, x_out=None, y_out=None):
        """x' = bf16(bf16(x W^T + b) + res) and y = LayerNorm(x'; ln = (gamma, beta)) in one launch
        (mx_gemm_bf16_res_ln): the residual Linear and the normalisation that reads its output. Only where
        res_ln_fits(M, N); returns (x', y)."""
        x2 = _rows(x, self.K)
        if x2.shape[1] != self.K:
            raise ValueError(f"input width {x2.shape[1]} != {self.K}")
        M, N = x2.shape[0], self.N
        r2 = _rows(res, N)
        X = x_out if x_out is not None else torch.empty(M, N, device=x2.device, dtype=BF)
        Y = y_out if y_out is not None else torch.empty(M, N, device=x2.device, dtype=BF)
        ws = RlnWorkspace.get(x2.device, N)
        _lib.check(_lib.load().mx_gemm_bf16_res_ln(
            stream(), x2.data_ptr(), x2.stride(0), self.w.data_ptr(), self.w.stride(0), ptr(self.b), r2.data_ptr(),
            r2.stride(0), X.data_ptr(), X.stride(0), ln[0].data_ptr(), ln[1].data_ptr(), Y.data_ptr(), Y.stride(0), M,
            N, self.K, self.Kw, float(eps), ws.stats.data_ptr(), ws.stats.numel(), ws.sync.data_ptr(),
            ws.sync.numel()), "mx_gemm_bf16_res_ln")
        return X, Y

    def res_rms(self, x, res, sc1, eps=1e-6, x_out=None, y_out=None):
        """x' = bf16(bf16(x W^T + b) + res) and y = the TRecViT RMSNorm of x' (sc1 = bf16(scale + 1)) in one launch
        (mx_gemm_bf16_res_rms). Only where res_ln_fits(M, N); returns (x', y)."""
        x2 = _rows(x, self.K)
        if x2.shape[1] != self.K:
            raise ValueError(f"input width {x2.shape[1]} != {self.K}")
        M, N = x2.shape[0], self.N
        r2 = _rows(res, N)
        X = x_out if x_out is not None else torch.empty(M, N, device=x2.device, dtype=BF)
        Y = y_out if y_out is not None else torch.empty(M, N, device=x2.device, dtype=BF)
        ws = RlnWorkspace.get(x2.device, N)
        _lib.check(_lib.load().mx_gemm_bf16_res_rms(
            stream(), x2.data_ptr(), x2.stride(0), self.w.data_ptr(), self.w.stride(0), ptr(self.b), r2.data_ptr(),
            r2.stride(0), X.data_ptr(), X.stride(0), sc1.data_ptr(), Y.data_ptr(), Y.stride(0), M, N, self.K, self.Kw,
            float(eps), ws.stats.data_ptr(), ws.stats.numel(), ws.sync.data_ptr(), ws.sync.numel()),
            "mx_gemm_bf16_res_rms")
        return X, Y


_TUNED_P = {}  # (M, N, Kw) -> (cfg, splits) of the split-K partial GEMM


def _partial(lin, cfg, sp, x2, P, M):
    return _lib.load().mx_gemm_bf16_partial(stream(), cfg, sp, x2.data_ptr(), x2.stride(0), lin.w.data_ptr(),
                                            lin.w.stride(0), P.data_ptr(), P.stride(1), P.stride(0), M, lin.N, lin.K,
                                            lin.Kw)


def has_partial_pick(M, lin):
    """Whether the split-K partial GEMM of (M, lin.N, lin.Kw) has a pick already (tuned in this process or in the
    fixed table), so that a caller under graph capture does not fall back to the untuned default."""
    key = (M, lin.N, lin.Kw)
    return key in _TUNED_P or (MxLin.use_table and key in _FIXED_P)


def _partial_cfg(lin, M, x2):
    """(cfg, splits) for the split-K partial GEMM: every config with a partial-sum mode x splits in 1..4 timed once on
    the real operands (outside graph capture), else 64x64 tiles with 2 splits."""
    key = (M, lin.N, lin.Kw)
    if key in _TUNED_P:
        return _TUNED_P[key]
    if MxLin.use_table and key in _FIXED_P:
        _TUNED_P[key] = _FIXED_P[key]
        return _TUNED_P[key]
    lib = _lib.load()
    best = (8, 2)
    if MxLin.autotune and not torch.cuda.is_current_stream_capturing():
        nk = lin.Kw // 64
        bt = float("inf")
        P = torch.empty(4, M, lin.N, device=x2.device, dtype=torch.float32)
        for cfg in range(lib.mx_gemm_ncfg()):
            for sp in (1, 2, 3, 4):
                if sp > 1 and (nk // sp < 2 or (sp - 1) * (-(-nk // sp)) >= nk):
                    continue
                run = lambda: _partial(lin, cfg, sp, x2, P, M)
                if run() != 0:
                    continue
                run()
                e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                e0.record()
                for _ in range(10):
                    run()
                e1.record()
                e1.synchronize()
                t = e0.elapsed_time(e1)
                if t < bt:
                    best, bt = (cfg, sp), t
        del P
    _TUNED_P[key] = best
    return best


def tune_gemm(lin, M, x2, y2, a, r2, ldr, r_rows, ws, reps=10):
    """Time every (tile config, split-K) candidate on the real operands; return the fastest. Runs eagerly on the
    current stream (writes y2, which the caller overwrites right after)."""
    lib = _lib.load()
    cands = []
    nk = lin.Kw // 64
    for cfg in range(lib.mx_gemm_ncfg()):
        for sp in ((1, 2, 3, 4, 6, 8) if tune_gemm.split_k else (1,)):
            if sp > 1 and (nk // sp < 3 or (sp - 1) * (-(-nk // sp)) >= nk):
                continue
            cands.append((cfg, sp))
        if tune_gemm.partial and a != 3:
            for sp in (2, 4, 8, 16):
                if nk // sp < 2 or (sp - 1) * (-(-nk // sp)) >= nk:
                    continue
                cands.append((cfg, -sp))
    best, bt = None, float("inf")
    for cfg, sp in cands:
        if sp > 1:
            ws.reserve(*_ws_need(cfg, sp, M, lin.N))
        elif sp < 0:
            ws.reserve(-sp * M * lin.N, 0)
        run = lambda: lin._launch(cfg, sp, x2, y2, M, a, r2, ldr, r_rows, ws)
        if run() != 0:
            continue
        run()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(reps):
            run()
        e1.record()
        e1.synchronize()
        t = e0.elapsed_time(e1)
        if t < bt:
            best, bt = (cfg, sp), t
    return best


# Split-K candidates in the tuner: off by default (the cross-XCD release fence of the last-arriver reduction costs
# more than the extra parallelism buys at these shapes; the path stays available and tested).
tune_gemm.split_k = False
# Fence-free split-K candidates (partial GEMM + mx_gemm_reduce, pick (cfg, -S)): on by default; they win where the
# grid of output tiles is far below the 256 CUs (the 32 / 64-row prompt and query GEMMs).
tune_gemm.partial = True


class MxI8Lin:
    """W8A8 Linear (the reference's HI8Lin, moondream/gpu/hgemm.py:95-137): int8 weights with a per-output-channel scale
    (amax / 127, round half to even, hgemm.py:101-106), int8 activations with a per-token dynamic scale (quant(),
    tgemm.py:81-91), int32 MFMA accumulation, fp32 dequant ((acc * s_x) * s_w) + bias, GELU-tanh on that fp32 value
    when asked (fused_gelu), one bf16 rounding (i8gemm.hip:181-197). `pre` takes an already quantised input (q, s),
    so layers that read the same activation share one quantisation (md2fast.py:52, 174). A residual is added to the
    rounded output and rounded again, exactly the reference's separate bf16 add (lin_res / mlp, md2fast.py:55-67),
    so the class also offers fused_res.
    Weights are zero-padded along K to a multiple of 128 (the int8 k-step); K must be a multiple of 16.
    """
    fused_gelu = True
    fused_res = True

    def __init__(self, weight, bias, dtype=BF, device="cuda"):
        assert dtype == BF, "bf16 activations only"
        w = weight.detach().to(device=device, dtype=BF)
        self.N, self.K = w.shape
        if self.K % 16 or self.N % 4:
            raise ValueError(f"W8A8 Linear needs K % 16 == 0 and N % 4 == 0, got {tuple(w.shape)}")
        self.Kw = (self.K + 127) // 128 * 128
        self.wq, self.sw = self.quantize_weight(w, self.Kw)
        self.b = None if bias is None else bias.detach().to(device=w.device, dtype=torch.float32).contiguous()
        self.cfgs = {}
        self.dev = w.device

    @classmethod
    def from_quantized(cls, wq, sw, bias):
        """A Linear over already quantised weights (int8 (N, Kw) with Kw % 128 == 0 and zeros past K = Kw, fp32 (N,)
        scales): row slices of a fused quantised weight share its storage."""
        self = cls.__new__(cls)
        self.N, self.Kw = wq.shape
        self.K = self.Kw
        if self.Kw % 128 or wq.stride(1) != 1 or wq.stride(0) % 16:
            raise ValueError("quantised weight rows must be contiguous, 16-byte aligned, a multiple of 128 wide")
        self.wq, self.sw = wq, sw
        self.b = None if bias is None else bias.detach().to(device=wq.device, dtype=torch.float32).contiguous()
        self.cfgs = {}
        self.dev = wq.device
        return self

    @staticmethod
    def quantize_weight(weight, Kw=None):
        """(N, K) bf16 weight (on the device) -> int8 (N, Kw) zero-padded past K, fp32 (N,) per-row scale
        (hgemm.py:101-106), by the library's quantisation kernel."""
        w = weight.detach().to(dtype=BF).contiguous()
        N, K = w.shape
        Kw = K if Kw is None else Kw
        q = torch.zeros(N, Kw, device=w.device, dtype=torch.int8)
        s = torch.empty(N, device=w.device, dtype=torch.float32)
        call("mx_quant_weight_i8", stream(), w.data_ptr(), w.stride(0), q.data_ptr(), q.stride(0), s.data_ptr(), N, K)
        return q, s

    def quant(self, x):
        """Per-token int8 quantisation of x (..., K) -> (q (M, K) int8, s (M,) fp32)."""
        x2 = _rows(x, self.K)
        M = x2.shape[0]
        q = torch.empty(M, self.K, device=x2.device, dtype=torch.int8)
        sc = torch.empty(M, device=x2.device, dtype=torch.float32)
        call("mx_quant_rows_i8", stream(), x2.data_ptr(), x2.stride(0), q.data_ptr(), q.stride(0), sc.data_ptr(), M,
             self.K)
        return q, sc

    def _launch(self, cfg, q, sc, y2, M, a, r2, ldr, r_rows, P=None, splits=1):
        """splits = -S: raw int32 partials of S splits into the workspace (mx_gemm_i8_partial), then the W8A8
        epilogue over their exact sum (mx_gemm_i8_reduce): equal to the one-launch GEMM bit for bit."""
        lib = _lib.load()
        if splits < 0:
            S, N = -splits, self.N
            ws = Workspace.get(q.device)
            if S * M * N > ws.ws.numel():
                return -3
            Pw = ws.ws[:S * M * N].view(torch.int32).view(S, M, N)
            rc = lib.mx_gemm_i8_partial(stream(), cfg, S, q.data_ptr(), q.stride(0), self.wq.data_ptr(),
                                        self.wq.stride(0), Pw.data_ptr(), N, M * N, M, N, self.K, self.Kw)
            if rc != 0:
                return rc
            return lib.mx_gemm_i8_reduce(stream(), Pw.data_ptr(), S, M * N, N, ptr(sc), self.sw.data_ptr(),
                                         ptr(self.b), ptr(r2), ldr, r_rows, y2.data_ptr(), y2.stride(0), M, N, a)
        return lib.mx_gemm_i8(stream(), cfg, q.data_ptr(), q.stride(0), self.wq.data_ptr(), self.wq.stride(0),
                              ptr(sc), self.sw.data_ptr(), ptr(self.b), ptr(r2), ldr, r_rows, ptr(y2),
                              y2.stride(0) if y2 is not None else 0, M, self.N, self.K, self.Kw, a, ptr(P),
                              P.stride(0) if P is not None else 0)

    def _pick(self, M, q, sc, y2):
        """(cfg, splits) for this M: every kind-0 tile config in one launch, and with raw partials over 2 / 4 / 8 / 16
        k-splits plus the reduction, each timed on the real operands (outside graph capture)."""
        key = ("i8", M, self.N, self.Kw)
        if key in _TUNED:
            return _TUNED[key]
        best = (0, 1)
        if MxLin.autotune and not torch.cuda.is_current_stream_capturing():
            bt = float("inf")
            nk = self.Kw // 128
            ws = Workspace.get(q.device)
            cands = [(c, 1) for c in range(_lib.load().mx_gemm_ncfg()) if _lib.load().mx_gemm_cfg_kind(c) == 0]
            if tune_gemm.partial:
                cands += [(c, -sp) for c, _ in list(cands) for sp in (2, 4, 8, 16)
                          if nk // sp >= 2 and (sp - 1) * (-(-nk // sp)) < nk]
            for cfg, sp in cands:
                if sp < 0:
                    ws.reserve(-sp * M * self.N, 0)
                run = lambda: self._launch(cfg, q, sc, y2, M, 0, None, 0, 0, splits=sp)
                if run() != 0:
                    continue
                run()
                e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                e0.record()
                for _ in range(5):
                    run()
                e1.record()
                e1.synchronize()
                t = e0.elapsed_time(e1)
                if t < bt:
                    best, bt = (cfg, sp), t
        _TUNED[key] = best
        return best

    def __call__(self, x, gelu=False, res=None, pre=None, act=None, out=None):
        a = ACT[act if act is not None else gelu]
        if a == 3:
            raise ValueError("no gated GELU in the W8A8 path")
        q, sc = pre if pre is not None else self.quant(x)
        M = q.shape[0]
        y = out if out is not None else torch.empty(M, self.N, device=q.device, dtype=BF)
        y2 = y.view(-1, self.N) if y.dim() != 2 else y
        r2, r_rows, ldr = None, 0, 0
        if res is not None:
            r2 = res.reshape(-1, self.N)
            if r2.stride(1) != 1:
                r2 = r2.contiguous()
            ldr = r2.stride(0)
            if r2.shape[0] != M:
                raise ValueError("residual rows must equal the output rows")
        cfg = self.cfgs.get(M)
        if cfg is None:
            cfg = self.cfgs[M] = self._pick(M, q, sc, y2)
        cfg, splits = cfg if isinstance(cfg, tuple) else (cfg, 1)
        if splits < 0:
            Workspace.get(q.device).reserve(-splits * M * self.N, 0)
        _lib.check(self._launch(cfg, q, sc, y2, M, a, r2, ldr, r_rows, splits=splits), "mx_gemm_i8")
        return y2.view(*x.shape[:-1], self.N) if out is None else y

    def acc_i32(self, q, cfg=0):
        """Raw int32 accumulators q Wq^T (M, N) (parity checks)."""
        M = q.shape[0]
        P = torch.empty(M, self.N, device=q.device, dtype=torch.int32)
        _lib.check(self._launch(cfg, q, None, None, M, 0, None, 0, 0, P=P), "mx_gemm_i8")
        return P


def sdpa(q, k, v, out=None, scale=None, qpos0=0, causal_from=None):
    """Fused attention. q (B, H, Tq, D), k/v (B, H, Tk, D) strided views (unit stride on D); out (B, Tq, H*D).

    Mask: key j is visible to query i iff j < Tk and (j < causal_from or j <= qpos0 + i); causal_from=None = no mask.
    """
    B, H, Tq, D = q.shape
    Tk = k.shape[2]
    if out is None:
        out = torch.empty(B, Tq, H * D, device=q.device, dtype=BF)
    sc = D ** -0.5 if scale is None else scale
    cf = Tk if causal_from is None else causal_from
    call("mx_sdpa", stream(), q.data_ptr(), q.stride(0), q.stride(1), q.stride(2),
         k.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.data_ptr(), v.stride(0), v.stride(1), v.stride(2),
         out.data_ptr(), out.stride(0), D, out.stride(1), B, H, Tq, Tk, D, float(sc), int(qpos0), int(cf))
    return out


def sdpa_tiling(B, H, Tq, D):
    """(query waves, key waves, keys per staged block, ring stages) of the kernel sdpa runs for this problem."""
    import ctypes
    t = (ctypes.c_int * 4)()
    _lib.load().mx_sdpa_tiling(B, H, Tq, D, ctypes.cast(t, ctypes.c_void_p))
    return tuple(t)


def sdpa_symbol(B, H, Tq, D):
    """The attention kernel's name as rocprofv3 prints it."""
    return "attn_fwd_kernel<{}, {}>".format(D, ", ".join(str(v) for v in sdpa_tiling(B, H, Tq, D)))


class Attn:
    """Reference protocol (hattn.py:17-37): Attn(H, T, D)(q, k, v) -> (B, T, H*D). No V^T staging buffer is needed:
    the kernel transposes V through LDS."""

    def __init__(self, H, T, D, device="cuda", scale=None):
        self.H, self.T, self.D = H, T, D
        self.scale = D ** -0.5 if scale is None else scale

    def __call__(self, q, k, v, out=None):
        return sdpa(q, k, v, out=out, scale=self.scale)


def layernorm(x, w, b, eps=1e-5, out=None):
    D = x.shape[-1]
    x2 = _rows(x, D)
    y = out if out is not None else torch.empty(x2.shape, device=x.device, dtype=BF)
    call("mx_layernorm", stream(), x2.data_ptr(), x2.stride(0), w.data_ptr(), b.data_ptr(), y.data_ptr(),
         y.reshape(-1, D).stride(0), x2.shape[0], D, float(eps))
    return y.view(*x.shape) if out is None else y


class RlnWorkspace:
    """Row statistics and their generation counters for mx_gemm_bf16_res_ln / _res_rms, one per (device, N), allocated
    zeroed once at their largest size (the launch allows at most one 64 x 64 tile per CU, so at most 256 tiles: 256
    x 128 stats words; 1 + 2 x 256 sync words) and then owned by the kernel, which leaves them ready for the next
    call. Keyed by N because where a row block's statistics sit depends on the tiles per row block (N / 64): calls
    of another N on the same words could meet old words that carry the epoch they expect. Calls of one N may have
    any M. Calls on one stream serialise; two streams must not share them."""
    _by_key = {}

    def __init__(self, device):
        self.stats = torch.zeros(256 * 128, device=device, dtype=torch.int64)
        self.sync = torch.zeros(1024, device=device, dtype=torch.int32)

    @staticmethod
    def _dev_index(device):
        d = torch.device(device)
        return d.index if d.index is not None else torch.cuda.current_device()

    @classmethod
    def get(cls, device, N):
        key = (cls._dev_index(device), int(N))
        if key not in cls._by_key:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the residual-LayerNorm workspace must exist before graph capture")
            cls._by_key[key] = cls(torch.device(device))
        return cls._by_key[key]

    @classmethod
    def device_error(cls, device):
        """Non-zero if a wait of any fused residual-LayerNorm GEMM on the device timed out (its results are then
        undefined). Synchronises."""
        i = cls._dev_index(device)
        return max((ws.error() for (d, _), ws in cls._by_key.items() if d == i), default=0)

    @classmethod
    def reset_device(cls, device):
        """Zero every workspace of the device (after a timed-out wait)."""
        i = cls._dev_index(device)
        for (d, _), ws in cls._by_key.items():
            if d == i:
                ws.reset()

    def error(self):
        """Non-zero if a wait of a fused residual-LayerNorm GEMM on these words timed out."""
        return int(self.sync[0].item())

    def reset(self):
        """Zero both buffers (after a timed-out wait, before the next call)."""
        self.stats.zero_()
        self.sync.zero_()


def _cu_count(device):
    return torch.cuda.get_device_properties(torch.device(device)).multi_processor_count


def res_ln_fits(M, N, device):
    """mx_gemm_bf16_res_ln's shape rule: N a multiple of 64 (at most 4096) and one 64 x 64 tile per CU at most."""
    return N % 64 == 0 and N <= 4096 and ((M + 63) // 64) * (N // 64) <= _cu_count(device)


def residual_layernorm(P, bias, res, ln=None, eps=1e-5, x_out=None, y_out=None):
    """Reduce split-K partials P (splits, M, D) fp32: x = bf16(bf16(sum P + bias) + res); y = LayerNorm(x; ln) when
    ln = (gamma, beta) is given. Returns (x, y) (y None without ln)."""
    S, M, D = P.shape
    r2 = _rows(res, D)
    x = x_out if x_out is not None else torch.empty(M, D, device=P.device, dtype=BF)
    y = None
    if ln is not None:
        y = y_out if y_out is not None else torch.empty(M, D, device=P.device, dtype=BF)
    call("mx_residual_layernorm", stream(), P.data_ptr(), S, P.stride(0), P.stride(1), ptr(bias), r2.data_ptr(),
         r2.stride(0), x.data_ptr(), x.stride(0), ptr(ln[0]) if ln else None, ptr(ln[1]) if ln else None, ptr(y),
         y.stride(0) if y is not None else 0, M, D, float(eps))
    return x, y


def residual_rmsnorm(P, bias, res, sc1, eps=1e-6, x_out=None, y_out=None):
    """Reduce split-K partials P (splits, M, D) fp32: x = bf16(bf16(sum P + bias) + res); y = the TRecViT RMSNorm of
    x with sc1 = bf16(scale + 1). Returns (x, y)."""
    S, M, D = P.shape
    r2 = _rows(res, D)
    x = x_out if x_out is not None else torch.empty(M, D, device=P.device, dtype=BF)
    y = y_out if y_out is not None else torch.empty(M, D, device=P.device, dtype=BF)
    call("mx_residual_rmsnorm", stream(), P.data_ptr(), S, P.stride(0), P.stride(1), ptr(bias), r2.data_ptr(),
         r2.stride(0), x.data_ptr(), x.stride(0), sc1.data_ptr(), y.data_ptr(), y.stride(0), M, D, float(eps))
    return x, y


def rmsnorm(x, sc1, eps=1e-6, out=None):
    """TRecViT RMSNorm; sc1 = bf16(scale + 1)."""
    D = x.shape[-1]
    x2 = _rows(x, D)
    y = out if out is not None else torch.empty(x2.shape, device=x.device, dtype=BF)
    call("mx_rmsnorm", stream(), x2.data_ptr(), x2.stride(0), sc1.data_ptr(), y.data_ptr(),
         y.reshape(-1, D).stride(0), x2.shape[0], D, float(eps))
    return y.view(*x.shape) if out is None else y


def patchify(img_u8, patch, mode, ldo=None, out=None):
    """(B, S, S, 3) u8 -> (B * (S/P)^2, ldo) bf16 patch rows, (c, ky, kx) column order, zero padded to ldo."""
    B, S, _, _ = img_u8.shape
    K = 3 * patch * patch
    ldo = (K + 7) // 8 * 8 if ldo is None else ldo
    G = S // patch
    y = out if out is not None else torch.empty(B * G * G, ldo, device=img_u8.device, dtype=BF)
    call("mx_patchify_u8", stream(), img_u8.data_ptr(), y.data_ptr(), ldo, B, S, patch, mode)
    return y


def resize_patchify(img_u8, size, patch, ldo=None, out=None):
    """(B, Hs, Ws, 3) u8 -> bilinear resize to size x size, / 127.5 - 1, as (B * (size/P)^2, ldo) bf16 patch rows
    (the TRecViT preprocess, tapnext/npu/step8.py:379-383, fused with the patch-conv input)."""
    B, Hs, Ws, _ = img_u8.shape
    K = 3 * patch * patch
    ldo = (K + 7) // 8 * 8 if ldo is None else ldo
    G = size // patch
    y = out if out is not None else torch.empty(B * G * G, ldo, device=img_u8.device, dtype=BF)
    call("mx_resize_patchify_u8", stream(), img_u8.data_ptr(), Hs, Ws, y.data_ptr(), ldo, B, size, patch)
    return y


# ------------------------------------------------------------------------------------------------ MXFP4, 8-bit KV cache
def _call_on(dev, name, *args):
    """call() on the current stream of the tensors' own device."""
    if dev.type != "cuda":
        raise ValueError(f"{name} needs tensors on the GPU, got {dev}")
    cur = torch._C._cuda_getDevice()  # a tensor is there, so the GPU is set up
    if dev.index == cur:
        rc = getattr(_lib._lib or _lib.load(), name)(torch._C._cuda_getCurrentRawStream(cur), *args)
        if rc:
            _lib.check(rc, name)
        return
    with torch.cuda.device(dev):
        call(name, stream(), *args)


def _need(t, name, dev, dtype=BF):
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{name} is on {t.device}, not on {dev}")


def _rows2(x):
    """2-D view (M, K) of x with unit column stride (copied if it has another)."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    return x if x.stride(1) == 1 or x.shape[1] == 1 else x.contiguous()


def _end(t):
    """The address behind the last element of a tensor that is not empty."""
    return t.data_ptr() + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size()


def _apart(a, b):
    """Whether the elements of a and b (the same type, neither empty) are known not to meet: they lie one behind the other, or
    side by side in the rows of one buffer."""
    if _end(a) <= b.data_ptr() or _end(b) <= a.data_ptr():
        return True
    pitch = b.stride(-2) if b.dim() > 1 else 0
    off, rest = divmod(b.data_ptr() - a.data_ptr(), b.element_size())
    if pitch < 1 or rest:
        return False
    wide = lambda t: 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()) if s % pitch)  # columns; other steps are rows
    return wide(a) <= off % pitch <= pitch - wide(b)


class MxFp4:
    """A matrix (rows, K) in MXFP4: 4-bit e2m1 codes and a power-of-two scale for each 32 columns of a row, in one buffer
    (uint8; the codes, then the scales, each in the order of the matrix instruction's operands)."""

    def __init__(self, data, rows, K):
        need = MxFp4.cells(rows, K) * 4352
        if rows < 0 or K < 1 or data.dtype != torch.uint8 or not data.is_contiguous() or data.numel() < need:
            raise ValueError(f"({rows}, {K}) in MXFP4 takes {need} contiguous uint8, got {tuple(data.shape)} {data.dtype}")
        if data.data_ptr() % 16:
            raise ValueError("data must be 16-byte aligned")
        self._hold(data, rows, K)

    def _hold(self, data, rows, K):
        self.data, self.rows, self.K = data, rows, K
        self.dev = data.device
        p = data.data_ptr()
        self.ptrs = p, p + MxFp4.cells(rows, K) * 4096  # codes, scales
        return self

    @staticmethod
    def cells(rows, K):
        """Pieces of 64 rows x 128 columns: 4 KB of codes and 256 bytes of scales each."""
        return (rows + 63) // 64 * ((K + 127) // 128)

    def values(self, out=None):
        """(rows, K) bf16: the values the codes stand for, exact."""
        dev, M, K = self.dev, self.rows, self.K
        if out is None:
            y = torch.empty(M, K, device=dev, dtype=BF)
        else:
            y = out
            _need(y, "out", dev)
            if y.shape != (M, K) or (y.stride(1) != 1 and K > 1):
                raise ValueError(f"out must be ({M}, {K}) with unit column stride")
        if M:
            _call_on(dev, "mx_mxfp4_values", *self.ptrs, y.data_ptr(), y.stride(0), M, K)
        return y


def quant_mxfp4(x):
    """x (..., K) bf16 -> MxFp4 of its rows. Per block of 32 columns e = max(floor(log2 max|x|) - 2, -127), codes
    e2m1(x 2^-e) to nearest even, saturating at 6 (OCP MX v1.0); a block with an infinity or NaN becomes NaN."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("x needs at least one column")
    _need(x, "x", x.device)
    x2 = _rows2(x)
    M, K = x2.shape
    buf = torch.empty(MxFp4.cells(M, K) * 4352, device=x.device, dtype=torch.uint8)
    q = MxFp4.__new__(MxFp4)._hold(buf, M, K)
    if M:
        _call_on(x.device, "mx_quant_mxfp4", x2.data_ptr(), x2.stride(0), *q.ptrs, M, K)
    return q


class MxFp4Lin:
    """MXFP4 Linear: y = act(x W^T + b) [+ res] with W quantised once and x per call (quant_mxfp4's rule for both), on the
    scaled MFMA; fp32 throughout, rounded to bf16 once. `pre` takes an already quantised input (MxFp4), so layers that
    read the same activation share one quantisation. Any (N, K); inputs have K columns, or K rounded up to 8 (Kp), of
    which the first K are read. act: None / "tanh" / "erf", on columns >= act_from. `out` may lie in the memory of x or res (res
    is copied first unless each of its elements is where its result goes). Few rows are quantised inside the product's
    launch; the results are the same."""
    fused_gelu = True
    fused_res = True

    def __init__(self, weight, bias, dtype=BF, device="cuda"):
        if dtype != BF:
            raise ValueError("bf16 activations only")
        if weight.dim() != 2:
            raise ValueError(f"weight must be (N, K), got {tuple(weight.shape)}")
        self._set(quant_mxfp4(weight.detach().to(device=device, dtype=BF)), bias)

    @classmethod
    def from_quantized(cls, w, bias):
        """A Linear over an already quantised (N, K) weight (MxFp4)."""
        self = cls.__new__(cls)
        self._set(w, bias)
        return self

    def _set(self, w, bias):
        self.wq, self.N, self.K = w, w.rows, w.K
        self.Kp = (w.K + 7) // 8 * 8  # the input width MxLin asks for
        self.dev = w.dev
        if self.N < 1:
            raise ValueError("the weight needs at least one row")
        if bias is not None and bias.shape != (self.N,):
            raise ValueError(f"bias must be ({self.N},)")
        self.b = None if bias is None else bias.detach().to(device=self.dev, dtype=torch.float32).contiguous()
        self.bp = ptr(self.b)
        self.rows, self.ln_cols = _lib.load().mx_gemv_mxfp4_rows(), _lib.load().mx_ln_gemv_mxfp4_cols()

    def quant(self, x):
        return quant_mxfp4(x)

    def __call__(self, x, gelu=False, res=None, pre=None, act=None, out=None, act_from=0):
        a = ACT[act if act is not None else gelu]
        if a == 3:
            raise ValueError("no gated GELU in the MXFP4 path")
        if act_from < 0:
            raise ValueError("act_from must not be negative")
        N, K = self.N, self.K
        if pre is None:
            if x.shape[-1] != K:
                if x.shape[-1] != self.Kp:
                    raise ValueError(f"input width {x.shape[-1]} != {K}")
                x = x[..., :K]
            _need(x, "x", self.dev)
            x2 = _rows2(x)
            M = x2.shape[0]
        else:
            if pre.K != K or pre.dev != self.dev:
                raise ValueError(f"pre: width {pre.K} on {pre.dev}, need {K} on {self.dev}")
            M = pre.rows
            if x is not None and x.numel() != M * x.shape[-1]:
                raise ValueError("x and pre have different rows")
        if out is None:
            y = y2 = torch.empty(M, N, device=self.dev, dtype=BF)
        else:
            y = out
            _need(y, "out", self.dev)
            y2 = y if y.dim() == 2 else y.view(-1, N)
            if y2.shape != (M, N) or (y2.stride(1) != 1 and N > 1):
                raise ValueError(f"out must be ({M}, {N}) with unit column stride")
        r2, r_rows, ldr = None, 0, 0
        if res is not None:
            _need(res, "res", self.dev)
            if res.shape[-1] != N:
                raise ValueError(f"residual width {res.shape[-1]} != {N}")
            r2 = _rows2(res)
            ldr = r2.stride(0)
            if r2.shape[0] != M:
                if not r2.shape[0] or M % r2.shape[0]:
                    raise ValueError("residual rows must equal or divide the output rows")
                r_rows = r2.shape[0]
            if M and out is not None and not _apart(r2, y2) and (
                    r_rows or r2.data_ptr() != y2.data_ptr() or (r2.stride(0) != y2.stride(0) and M > 1)):
                # only where every element of res lies in the place of its own result may the product write over it
                r2 = r2.clone(memory_format=torch.contiguous_format)
                ldr = r2.stride(0)
        if M:
            tail = (*self.wq.ptrs, self.bp, None if r2 is None else r2.data_ptr(), ldr, r_rows, y2.data_ptr(), y2.stride(0), M, N, K, a, act_from)
            if pre is None and M <= self.rows and (out is None or _apart(x2, y2)):
                _call_on(self.dev, "mx_gemv_mxfp4", x2.data_ptr(), x2.stride(0), *tail)
            else:
                q = quant_mxfp4(x2) if pre is None else pre
                _call_on(self.dev, "mx_gemm_mxfp4", *q.ptrs, *tail)
        if out is not None or x is None or x.dim() == 2:
            return y
        return y.view(*x.shape[:-1], N)


    def ln(self, x, ln, eps=1e-5, act=None, out=None, act_from=0):
        """layernorm(x, *ln, eps) through the Linear: the same result; one row of at most 2048 columns (a multiple of 8) is
        normalised inside the product's launch."""
        N, K = self.N, self.K
        if x.shape[-1] != K or any(t.shape != (K,) or not t.is_contiguous() for t in ln):
            raise ValueError(f"x (..., {K}) and two contiguous ({K},) vectors, got {tuple(x.shape)}, {[tuple(t.shape) for t in ln]}")
        for t, name in ((x, "x"), (ln[0], "gamma"), (ln[1], "beta")):
            _need(t, name, self.dev)
        if x.numel() != K or K % 8 or K > self.ln_cols:
            if self.dev.type != "cuda":
                raise ValueError(f"ln needs tensors on the GPU, got {self.dev}")
            with torch.cuda.device(self.dev):
                return self(layernorm(x, *ln, eps=eps), act=act, out=out, act_from=act_from)
        a = ACT[act]
        if a == 3 or act_from < 0:
            raise ValueError("no gated GELU in the MXFP4 path, and act_from must not be negative")
        x2 = _rows2(x)
        y = torch.empty(1, N, device=self.dev, dtype=BF) if out is None else out
        _need(y, "out", self.dev)
        y2 = y if y.dim() == 2 else y.view(-1, N)
        if y2.shape != (1, N) or (y2.stride(1) != 1 and N > 1):
            raise ValueError(f"out must be (1, {N}) with unit column stride")
        if not _apart(x2, y2):
            x2 = x2.clone()
        _call_on(self.dev, "mx_ln_gemv_mxfp4", x2.data_ptr(), ln[0].data_ptr(), ln[1].data_ptr(), float(eps), *self.wq.ptrs,
                 self.bp, y2.data_ptr(), N, K, a, act_from)
        return y if out is not None or x.dim() == 2 else y.view(*x.shape[:-1], N)


def mxfp4_tiling(M, N, K):
    """(rows, columns per workgroup, ring steps (0: the few-row kernel), waves) of the product of M quantised rows."""
    import ctypes
    t = (ctypes.c_int * 4)()
    _lib.load().mx_gemm_mxfp4_tiling(M, N, K, ctypes.cast(t, ctypes.c_void_p))
    return tuple(t)


def _where(v, B, dev, name):
    """(pointer, stride, value) of a position or length: an int, or an int32 tensor of B values."""
    if isinstance(v, torch.Tensor):
        if v.dim() != 1 or v.shape[0] != B:
            raise ValueError(f"{name} must be an int or a tensor of {B} values")
        _need(v, name, dev, torch.int32)
        return v.data_ptr(), v.stride(0), 0
    return None, 0, int(v)


def _int32(v, name):
    if not -0x80000000 <= v <= 0x7fffffff:
        raise ValueError(f"{name} {v} does not fit 32 bits")
    return v


def _steps(t):
    """The strides of t, 0 for dimensions of size 1: what those carry is never walked."""
    return [s if n > 1 else 0 for n, s in zip(t.shape, t.stride())]


def _rows4(t):
    """t with unit column stride (copied if it has another)."""
    return t if t.stride(-1) == 1 else t.contiguous()


class KV8Cache:
    """A KV cache in 8 bits: e4m3 codes, one power-of-two scale for each block of 64 tokens of a head, K and V apart.
    `slots` sequences of at most `ctx` tokens, `heads` key heads of dim 64 or 128, contiguous per sequence. What the cache
    holds is exact in bf16 (read(); but for what rounds to 2^128); the codes are stored in the order of the matrix instruction's operands.
    Calls on one cache belong on one stream (or must be ordered by the caller), as with any tensor that is written."""
    BLOCK = 64

    def __init__(self, slots, heads, ctx, hd, device="cuda"):
        if min(slots, heads, ctx) < 1 or hd not in (64, 128):
            raise ValueError(f"slots {slots}, heads {heads}, ctx {ctx} must be positive and hd {hd} be 64 or 128")
        self.slots, self.heads, self.ctx, self.hd = slots, heads, ctx, hd
        nb = -(-ctx // self.BLOCK)
        z = lambda *s: torch.zeros(*s, device=device, dtype=torch.uint8)
        self._hold(z(slots, heads, nb, 64 * hd), z(slots, heads, nb, 64 * hd), z(slots, heads, nb), z(slots, heads, nb))

    @classmethod
    def over(cls, kc, vc, ks, vs, ctx):
        """A cache of ctx tokens over given storage (uint8, contiguous, zero at first): codes (slots, heads, blocks, 64 *
        hd) and scales (slots, heads, blocks) of ceil(ctx / 64) blocks."""
        slots, heads, nb, w = kc.shape
        self = cls.__new__(cls)
        self.slots, self.heads, self.ctx, self.hd = slots, heads, ctx, w // 64
        if nb < 1 or nb != -(-ctx // cls.BLOCK) or w not in (64 * 64, 64 * 128):
            raise ValueError(f"codes {tuple(kc.shape)} do not hold {ctx} tokens of head dim 64 or 128")
        for t, shape in ((kc, kc.shape), (vc, kc.shape), (ks, kc.shape[:3]), (vs, kc.shape[:3])):
            if t.shape != shape or t.dtype != torch.uint8 or not t.is_contiguous() or t.device != kc.device:
                raise ValueError("storage must be contiguous uint8 tensors of matching shapes on one device")
        if kc.data_ptr() % 16 or vc.data_ptr() % 16:
            raise ValueError("codes must be 16-byte aligned")
        self._hold(kc, vc, ks, vs)
        return self

    def _hold(self, kc, vc, ks, vs):
        self.kc, self.vc, self.ks, self.vs, self.dev = kc, vc, ks, vs, kc.device
        self.ptrs = kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr()
        self._ws = {}  # workspace floats of an attention call by (sequences, group, queries)

    def append(self, k, v, pos=0, base=0, count=None, bcast=False, cs=None, q=None):
        """Writes k, v (B, heads, n, hd) at positions base + pos_b + t of slot b (bcast: B = 1, into every slot). pos: an
        int, or an int32 tensor (B,) read on the device, so that a captured graph follows it; rows whose position then
        falls outside the cache are dropped (with an int that raises). count (int32 tensor (B,)): only the first
        count[b] rows of sequence b. A block that already holds rows before pos_b keeps its exponent or raises it (its
        codes are rounded to the new one). The sequence then ends behind the new rows: what their last block holds after
        them is undefined, other blocks and slots stay as they are.
        cs: the rotary table (positions, 16, 2) of synth.freqs_cis, hd = 64 only: k is rotated first, and q (B, Hq, n, hd)
        with it, which is returned as (B, Hq, n, hd)."""
        if k.dim() != 4 or k.shape != v.shape or k.shape[1] != self.heads or k.shape[3] != self.hd:
            raise ValueError(f"k, v must be (B, {self.heads}, n, {self.hd}), got {tuple(k.shape)}, {tuple(v.shape)}")
        B, H, n, D = k.shape
        if (B != 1) if bcast else (B > self.slots):
            raise ValueError(f"{B} sequences for {'a broadcast' if bcast else self.slots}")
        _need(k, "k", self.dev)
        _need(v, "v", self.dev)
        pp, ps, p0 = _where(pos, B, self.dev, "pos")
        base = _int32(int(base) + p0, "base")
        if pp is None and not 0 <= base <= self.ctx - n:
            raise ValueError(f"positions {base} .. {base + n - 1} outside the {self.ctx}-entry cache")
        cp, cstr, _ = (None, 0, 0) if count is None else _where(count, B, self.dev, "count")
        if count is not None and cp is None:
            raise ValueError("count must be a tensor")
        q_out, qa = None, (None, 0, 0, 0, 0, None)
        if q is not None and cs is None:
            raise ValueError("q goes with cs")
        if cs is not None:
            _need(cs, "cs", self.dev, torch.float32)
            if D != 64 or cs.dim() != 3 or cs.shape[1:] != (16, 2) or cs.shape[0] < 1 or not cs.is_contiguous():
                raise ValueError("cs must be a contiguous (positions, 16, 2) table and hd 64")
            if pp is None and base + n > cs.shape[0]:
                raise ValueError(f"position {base + n - 1} is past the {cs.shape[0]}-entry rotary table")
            if q is not None:
                if q.dim() != 4 or q.shape[0] != B or q.shape[2:] != k.shape[2:]:
                    raise ValueError(f"q must be ({B}, Hq, {n}, {D}), got {tuple(q.shape)}")
                _need(q, "q", self.dev)
                q = _rows4(q)
                q_out = torch.empty(q.shape, device=self.dev, dtype=BF)
                qa = (q.data_ptr(), *q.stride()[:3], q.shape[1], q_out.data_ptr())
        if k.numel():
            k, v = _rows4(k), _rows4(v)
            _call_on(self.dev, "mx_kv8_append", k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3],
                     *self.ptrs, B, H, n, D, self.ctx, self.slots, int(bcast), pp, ps, base, cp, cstr, ptr(cs),
                     0 if cs is None else cs.shape[0], *qa)
        return q_out

    def reorder(self, parent, n=None, first=0):
        """Slot g W + w becomes a copy of slot g W + parent[g, w] (reorder_slots, unit 64), over blocks first // 64 .. ceil(n / 64)
        - 1: tokens before `first` in its block go along. Four launches."""
        for t in (self.kc, self.vc, self.ks, self.vs):
            reorder_slots(t[None], parent, n, first, self.BLOCK)

    def read(self, n=None):
        """(k, v), each (slots, heads, n, hd) bf16: what positions 0 .. n - 1 (default: all) hold, exact."""
        n = self.ctx if n is None else int(n)
        if not 0 <= n <= self.ctx:
            raise ValueError(f"n {n} outside 0 .. {self.ctx}")
        k = torch.empty(self.slots, self.heads, n, self.hd, device=self.dev, dtype=BF)
        v = torch.empty_like(k)
        if n:
            _call_on(self.dev, "mx_kv8_read", *self.ptrs, k.data_ptr(), v.data_ptr(), self.slots, self.heads, n, self.hd,
                     self.ctx)
        return k, v


def sdpa_kv8(q, cache, kv_len, base=0, out=None, scale=None, qpos0=None, causal_from=None):
    """Attention of q (B, Hq, Tq, D) over the first base + kv_len_b tokens of slots 0 .. B - 1 of a KV8Cache, Hq a multiple
    of its heads (query head h reads key head h / (Hq / heads)); out (B, Tq, Hq * D).

    kv_len: an int, or an int32 tensor (B,) read on the device (values outside 0 .. ctx are clamped). Mask, as in sdpa:
    key j is visible to query i iff j < len_b and (j < causal_from or j <= qpos0 + i); causal_from=None: no mask;
    qpos0=None: the queries are the last Tq tokens of their sequence, qpos0 = len_b - Tq. Rows that see no key are 0.
    out may lie in q's memory.
    Scores (times scale) have to stay below 2^29 in size: larger ones come out as 0 or NaN.
    q and the softmax weights are taken in 8 bits (two e4m3 terms); sums of weights are fp32. The keys are cut into runs by the
    cache's ctx, not by the lengths: one token over a cache much longer than its sequence takes up to 2.5 times as long."""
    if q.dim() != 4 or q.shape[3] != cache.hd or q.shape[1] < 1 or q.shape[1] % cache.heads or q.shape[0] > cache.slots:
        raise ValueError(f"q {tuple(q.shape)} does not fit a cache of {cache.slots} x {cache.heads} heads x {cache.hd}")
    B, Hq, Tq, D = q.shape
    dev = cache.dev
    _need(q, "q", dev)
    lp, ls, l0 = _where(kv_len, B, dev, "kv_len")
    base = _int32(int(base) + l0, "base")
    if lp is None and not 0 <= base <= cache.ctx:
        raise ValueError(f"length {base} outside the {cache.ctx}-entry cache")
    sc = D ** -0.5 if scale is None else float(scale)
    if not 0.0 < sc <= 2.0 ** 127:  # the kernel multiplies by scale log2(e), a float
        raise ValueError(f"scale {sc} must be positive and finite, at most 2^127")
    cf = 0x7fffffff if causal_from is None else min(int(causal_from), 0x7fffffff)
    if cf < 0:
        raise ValueError("causal_from must not be negative")
    q0 = 0 if qpos0 is None else max(-0x80000000, min(int(qpos0), 0x7fffffff))  # positions all lie inside 31 bits
    given = out is not None
    if not given:
        out = torch.empty(B, Tq, Hq * D, device=dev, dtype=BF)
        so = out.stride()
    else:
        _need(out, "out", dev)
        so = _steps(out)
        if out.shape != (B, Tq, Hq * D) or so[2] != 1 or (so[0] | so[1]) % 4 or out.data_ptr() % 8:
            raise ValueError(f"out must be ({B}, {Tq}, {Hq * D}) with 8-byte aligned rows of unit stride")
    if not out.numel():
        return out
    if given and not _apart(q, out):
        q = q.clone()  # a row's output may lie over another's query
    s = _steps(q)
    if s[3] != 1 or (s[0] | s[1] | s[2]) % 8 or q.data_ptr() % 16:
        q = q.contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        s = _steps(q)
    G = Hq // cache.heads
    need = cache._ws.get((B, G, Tq))
    if need is None:
        need = cache._ws[(B, G, Tq)] = _lib.load().mx_kv8_sdpa_ws(B, cache.heads, G, Tq, cache.ctx, D)
    part = torch.empty(need, device=dev, dtype=torch.float32) if need else None
    _call_on(dev, "mx_kv8_sdpa", q.data_ptr(), s[0], s[1], s[2], *cache.ptrs, out.data_ptr(), so[0], so[1],
             B, cache.heads, G, Tq, D, cache.ctx, lp, ls, base, q0, int(qpos0 is None), cf, sc, ptr(part), need)
    return out


def sdpa_kv8_tiling(B, heads, G, Tq, ctx, hd):
    """(rows per workgroup (16: the few-row kernel), waves that share the keys, runs of keys, blocks per run) of sdpa_kv8 for B
    sequences, G query heads per key head, in a cache of ctx positions."""
    import ctypes
    t = (ctypes.c_int * 4)()
    _lib.load().mx_kv8_sdpa_tiling(B, heads, G, Tq, ctx, hd, ctypes.cast(t, ctypes.c_void_p))
    return tuple(t)


# ------------------------------------------------------------------------------------------------ shared prefixes, beams
class _PrefixCall:
    """A checked geometry of sdpa_prefix (shapes, strides and a device; nothing of the data)."""

    def __init__(self, q, pk, pv, k, v):
        if q.dim() != 4 or pk.dim() != 4 or pk.shape != pv.shape or k.dim() != 4 or k.shape != v.shape:
            raise ValueError(f"q, pk, pv, k, v: {tuple(q.shape)}, {tuple(pk.shape)}, {tuple(pv.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
        B, Hq, Tq, D = q.shape
        N, H, P = pk.shape[:3]
        if D not in (64, 128) or N < 1 or H < 1 or B % N or Hq % H or Hq < 1:
            raise ValueError(f"{B} sequences of {Hq} heads of dim {D} over {N} prefixes of {H} heads")
        if pk.shape[3] != D or k.shape[0] != B or k.shape[1] != H or k.shape[3] != D:
            raise ValueError(f"keys must be ({N}, {H}, P, {D}) and ({B}, {H}, T, {D}), got {tuple(pk.shape)}, {tuple(k.shape)}")
        for t, name in ((q, "q"), (pk, "pk"), (pv, "pv"), (k, "k"), (v, "v")):
            _need(t, name, q.device)
        self.dev, self.N, self.P, self.T, self.B = q.device, N, P, k.shape[2], B
        self.out = (B, Tq, Hq * D)
        self.sizes = (N, B // N, H, Hq // H, Tq, D, P, self.T)
        if max(self.sizes) > 0x7fffffff:
            raise ValueError(f"q {tuple(q.shape)}, pk {tuple(pk.shape)}, k {tuple(k.shape)}: the sizes do not fit 32 bits")
        self.work = B * Tq > 0
        self.scale = D ** -0.5
        # which have to be copied before the kernel takes them: rows that are not of unit stride, 16-byte steps and 31-bit offsets
        steps = [_steps(t) for t in (q, pk, pv, k, v)]
        self.odd = [s[3] != 1 or (s[0] | s[1] | s[2]) % 8 != 0 or (i > 0 and not 0 <= s[2] < 0x800000) for i, s in enumerate(steps)]
        self.copy = any(self.odd)
        self.need = 0
        if self.work:
            import ctypes
            self.strides = (ctypes.c_long * 15)(*(x for s in steps for x in s[:3]))
            self.need = _lib.load().mx_sdpa_prefix_ws(N, B // N, H, Hq // H, Tq, P, self.T, D)


_PREFIX_CALLS = {}


def sdpa_prefix(q, pk, pv, k, v, kv_len=None, prefix_len=None, out=None, scale=None, causal=True):
    """Attention of sequences that share prefixes: q (B, Hq, Tq, D), prefixes pk, pv (N, H, P, D), own keys k, v (B, H, T, D); D 64
    or 128, Hq a multiple of H (query head h reads key head h / (Hq / H)), B of N: sequence b has prefix b // (B / N), which is
    stored once for all of them. Returns out (B, Tq, Hq * D).

    How often keys are read: a workgroup reads those of its rows, so the prefix goes through the caches once for every 16 to 128
    rows (sequence, query, head of a group) where a sequence has fewer than 32 rows per key head, of any sequences of the prefix,
    and once for every 32 to 256 rows of one sequence else (sdpa_prefix_tiling).

    Query i sees keys 0 .. prefix_len_n - 1 of its prefix and, of its own first kv_len_b keys, those up to its own: the queries
    are the sequence's last Tq tokens, key t is visible iff t <= kv_len_b - Tq + i (causal=False: all kv_len_b). A row that sees
    no key is 0. kv_len, prefix_len: an int, or an int32 tensor (B,) / (N,) read on the device (clamped to 0 .. T / 0 .. P);
    None: all. out may lie in q's memory, not in the keys' or values'. Scores (times scale) have to stay below 2^29 in size, N S H
    below 2^23 and N S H G Tq below 2^24 (S sequences of a prefix, G query heads of a key head). Keys that a row does not see may
    hold infinities and NaN; an infinite value of one that it sees gives the formula's infinity or NaN, and either of them where
    its weight underflows to 0."""
    key = (q.shape, q.stride(), pk.shape, pk.stride(), pv.shape, pv.stride(), k.shape, k.stride(), v.shape, v.stride(), q.device)
    c = _PREFIX_CALLS.get(key)
    if c is None or not (q.dtype is BF and pk.dtype is BF and pv.dtype is BF and k.dtype is BF and v.dtype is BF and
                         q.device == pk.device == pv.device == k.device == v.device):
        c = _PrefixCall(q, pk, pv, k, v)
        if len(_PREFIX_CALLS) >= 4096:  # a program of ever new lengths
            _PREFIX_CALLS.clear()
        _PREFIX_CALLS[key] = c
    dev = c.dev
    lp, ls, l0 = (None, 0, c.T) if kv_len is None else _where(kv_len, c.B, dev, "kv_len")
    pp, ps, p0 = (None, 0, c.P) if prefix_len is None else _where(prefix_len, c.N, dev, "prefix_len")
    if not 0 <= l0 <= c.T or not 0 <= p0 <= c.P:
        raise ValueError(f"kv_len {l0} of {c.T} keys, prefix_len {p0} of {c.P}")
    sc = c.scale
    if scale is not None:
        sc = float(scale)
        if not 0.0 < sc <= 2.0 ** 127:  # the kernel multiplies by scale log2(e), a float
            raise ValueError(f"scale {sc} must be positive and finite, at most 2^127")
    given = out is not None
    if not given:
        out = torch.empty(c.out, device=dev, dtype=BF)
        so = c.out[1] * c.out[2], c.out[2]
    else:
        _need(out, "out", dev)
        so = _steps(out)
        if out.shape != c.out or so[2] != 1 or (so[0] | so[1]) % 4 or out.data_ptr() % 8:
            raise ValueError(f"out must be {c.out} with 8-byte aligned rows of unit stride")
    if not c.work:
        return out
    if given and not _apart(q, out):
        q = q.clone(memory_format=torch.contiguous_format)  # a row's output may lie over another's query
        return sdpa_prefix(q, pk, pv, k, v, kv_len, prefix_len, out, scale, causal)
    qp, pkp, pvp, kp, vp = q.data_ptr(), pk.data_ptr(), pv.data_ptr(), k.data_ptr(), v.data_ptr()
    if c.copy or (qp | pkp | pvp | kp | vp) & 15:
        q, pk, pv, k, v = (t.clone(memory_format=torch.contiguous_format) if odd or t.data_ptr() & 15 else t
                           for t, odd in zip((q, pk, pv, k, v), c.odd))
        return sdpa_prefix(q, pk, pv, k, v, kv_len, prefix_len, out, scale, causal)
    need = c.need
    part = torch.empty(need, device=dev, dtype=torch.float32) if need else None
    _call_on(dev, "mx_sdpa_prefix", qp, pkp or None, pvp or None, kp or None, vp or None, out.data_ptr(), c.strides, so[0], so[1],
             *c.sizes, pp, ps, p0, lp, ls, l0, 1 if causal else 0, sc, part.data_ptr() if need else None, need)
    return out


def sdpa_prefix_tiling(N, S, heads, G, Tq, P, T, hd):
    """How sdpa_prefix cuts N prefixes of S sequences each, G query heads per key head: (0 rows / 1 both / 2 tiles, query and key
    waves and runs of the tile kernel, rows per workgroup and runs of the few-row kernel)."""
    import ctypes
    t = (ctypes.c_int * 6)()
    sizes = [_int32(v, "size") for v in (N, S, heads, G, Tq, P, T, hd)]
    _lib.load().mx_sdpa_prefix_tiling(*sizes, ctypes.cast(t, ctypes.c_void_p))
    return tuple(t)


_SELECT_CALLS = {}


def _select_call(logits, scores, k, done, eos):
    """(k, eos or -1, bytes of workspace, whether the logits' columns have to be gathered) of a checked geometry."""
    if logits.dim() != 3 or logits.dtype not in (BF, torch.float32):
        raise ValueError(f"logits must be (B, W, V) in bf16 or fp32, got {tuple(logits.shape)} {logits.dtype}")
    B, W, V = logits.shape
    k = W if k is None else k
    if not (1 <= W <= 64 and 1 <= k <= 64 and V >= 1):
        raise ValueError(f"{W} beams over {V} tokens, {k} to select: at most 64 of each, at least 1")
    if max(B, V) > 0x7fffffff:
        raise ValueError(f"logits {tuple(logits.shape)}: the sizes do not fit 32 bits")
    _need(scores, "scores", logits.device, torch.float32)
    if scores.shape != (B, W):
        raise ValueError(f"scores must be ({B}, {W}), got {tuple(scores.shape)}")
    e = -1 if eos is None else eos
    if eos is not None and not 0 <= e < V:
        raise ValueError(f"eos {e} outside the {V} tokens")
    if done is not None:
        if eos is None:
            raise ValueError("done goes with eos")
        _need(done, "done", logits.device, torch.bool)
        if done.shape != (B, W):
            raise ValueError(f"done must be ({B}, {W}), got {tuple(done.shape)}")
    need = _lib.load().mx_beam_select_ws(max(B, 1), W, V, k)
    if not need:
        raise ValueError(f"{B} x {W} beams over {V} tokens, {k} to select: too many")
    return k, e, need, logits.stride(2) != 1 and V > 1


def beam_select(logits, scores, k=None, done=None, eos=None):
    """Beam search's selection: logits (B, W, V) bf16 or fp32 of W beams with scores (B, W) fp32. Returns (score, parent, token,
    done), each (B, k) (k: default W): the k largest of scores[b, w] + log_softmax(logits[b, w])[v] in falling order, equal ones
    by the lowest beam, then the lowest token; parent = w, token = v (int32). Within a beam the order is exact; between beams it is
    that of the computed values, whose sums of exponentials are fp32 within 8192 logits: two that lie nearer than 2^-17 may come
    in either order.

    A finished beam (done (B, W) bool) offers eos alone, at its score; the returned done says which hypotheses end in eos (None
    without eos). A beam whose score is not finite, or whose logits hold NaN or +infinity or nothing above -infinity, offers
    nothing, and neither does a logit of -infinity (a score of -infinity, say, keeps the copies of a first beam out). Places that
    are left hold score -infinity, parent 0, token eos (0 without), done. W and k at most 64, B below 2^22, V as far as a search's
    lists of candidates fit the LDS (350000 for the largest W and k, millions for the usual ones)."""
    # (numbers, never a tensor that holds one: the geometry is kept by them)
    k, eos = None if k is None else int(k), None if eos is None else int(eos)
    key = (logits.shape, logits.stride(), logits.dtype, logits.device, scores.shape, scores.dtype, scores.device, k, eos,
           None if done is None else (done.shape, done.dtype, done.device))
    c = _SELECT_CALLS.get(key)
    if c is None:
        c = _select_call(logits, scores, k, done, eos)
        if len(_SELECT_CALLS) >= 4096:
            _SELECT_CALLS.clear()
        _SELECT_CALLS[key] = c
    k, e, n, gather = c
    B, W, V = logits.shape
    dev = logits.device
    if gather:
        logits = logits.contiguous()
    score = torch.empty(B, k, device=dev, dtype=torch.float32)
    parent = torch.empty(B, k, device=dev, dtype=torch.int32)
    token = torch.empty(B, k, device=dev, dtype=torch.int32)
    od = None if e < 0 else torch.empty(B, k, device=dev, dtype=torch.bool)
    if B:
        ws = torch.empty(n, device=dev, dtype=torch.uint8)
        scores = scores.contiguous()
        if done is not None:
            done = done.contiguous()
        s = logits.stride()
        _call_on(dev, "mx_beam_select", logits.data_ptr(), 0 if logits.dtype is BF else 1, s[0], s[1], scores.data_ptr(),
                 None if done is None else done.data_ptr(), e, B, W, V, k, score.data_ptr(), parent.data_ptr(), token.data_ptr(),
                 None if od is None else od.data_ptr(), ws.data_ptr(), n)
    return score, parent, token, od


def _disjoint(t):
    """Whether no two elements of t share memory (by its strides, largest last; sufficient)."""
    end = 1
    for s, n in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if s < end:
            return False
        end = s * (n - 1) + end
    return True


def reorder_slots(x, parent, n=None, first=0, unit=1):
    """Reorders the slots of a cache in place: x (L, slots, H, T, ...), whose rows x[l, s, h, t] are contiguous, any type; parent
    (G, W) int32, G W = slots (or (slots,)): slot g W + w becomes a copy of slot g W + parent[g, w], which may be any of its group,
    several times the same; values outside 0 .. W - 1 leave their slot. Only rows first .. n - 1 move, n an int or an int32 tensor
    (slots,) of the rows that each slot holds (a slot takes as many as its parent has; None: all T); every other row stays. unit:
    tokens per row; first and n then count tokens, and rows first // unit .. ceil(n / unit) - 1 move. W at most 64; T, n and the
    bytes of a row below 2^31. Rows move in pieces of 16 bytes, of 4 where an address or a stride is no multiple of 16, or of
    1; a call takes L G H ceil(pieces of a slot's rows / 256) below 2^23. Returns x."""
    if x.dim() < 4:
        raise ValueError(f"x must be (L, slots, H, T, ...), got {tuple(x.shape)}")
    N, S, H, T = x.shape[:4]
    dev = x.device
    _need(parent, "parent", dev, torch.int32)
    if parent.dim() == 1:
        parent = parent[None]
    if parent.dim() != 2 or parent.numel() != S or not 1 <= parent.shape[1] <= 64:
        raise ValueError(f"parent must be (G, W) with G W = {S} and W at most 64, got {tuple(parent.shape)}")
    G, W = parent.shape
    first, unit = int(first), _int32(unit, "unit")
    if first < 0 or unit < 1:
        raise ValueError(f"first {first} must not be negative, unit {unit} at least 1")
    lp, ls, l0 = _where(T * unit if n is None else n, S, dev, "n")
    if not 0 <= l0 <= T * unit:
        raise ValueError(f"n {l0} outside 0 .. {T * unit}")
    if not x.is_contiguous():
        if not _disjoint(x) or (x.dim() > 4 and not x[0, 0, 0, 0].is_contiguous()):
            raise ValueError("x must not overlap itself, and its rows must be contiguous")
    cells = N * S * H * T
    if cells and x.numel():
        es, s = x.element_size(), x.stride()
        row = x.numel() // cells * es
        if max(N, S, H, T, row) > 0x7fffffff:
            raise ValueError(f"x {tuple(x.shape)}: its sizes and a row's {row} bytes do not fit 32 bits")
        _call_on(dev, "mx_reorder_slots", x.data_ptr(), s[0] * es, s[1] * es, s[2] * es, s[3] * es, N, G, W, H, T,
                 row, parent.data_ptr(), *parent.stride(), lp, ls, _int32(l0, "n"), unit, min(first // unit, T))
    return x


def rope_kv_at(qkv, cs, kc, vc, at, rot0=0):
    """The text decoder's rotary embedding and K / V write for rows whose place is on the device: qkv (B, n, >= 3 H 64) fused rows
    (q | k | v), cs the (positions, 16, 2) table, caches kc, vc (B, H, ctx, 64). Row t of sequence b is written at cache row
    at[b] + t (int32) and rotated for position rot0 + at[b] + t; rows outside the cache or the table are dropped. Returns the
    rotated q (B, H, n, 64)."""
    if kc.dim() != 4 or kc.shape != vc.shape or kc.shape[3] != 64 or qkv.dim() != 3 or qkv.shape[0] != kc.shape[0]:
        raise ValueError(f"qkv {tuple(qkv.shape)}, caches {tuple(kc.shape)}, {tuple(vc.shape)}: need (B, n, 3 H 64), (B, H, ctx, 64)")
    B, H, ctx = kc.shape[:3]
    n, dev = qkv.shape[1], qkv.device
    _need(qkv, "qkv", dev)
    _need(kc, "kc", dev)
    _need(vc, "vc", dev)
    _need(cs, "cs", dev, torch.float32)
    _need(at, "at", dev, torch.int32)
    if cs.dim() != 3 or cs.shape[1:] != (16, 2) or cs.shape[0] < 1 or not cs.is_contiguous():
        raise ValueError("cs must be a contiguous (positions, 16, 2) table")
    if max(B, n, H, ctx, cs.shape[0]) > 0x7fffffff:
        raise ValueError(f"qkv {tuple(qkv.shape)}, caches {tuple(kc.shape)}, {cs.shape[0]} positions: the sizes do not fit 32 bits")
    if at.shape != (B,) or not kc.is_contiguous() or not vc.is_contiguous() or qkv.shape[2] < 3 * H * 64:
        raise ValueError(f"at must be ({B},), the caches contiguous, qkv rows {3 * H * 64} wide")
    q = torch.empty(B, H, n, 64, device=dev, dtype=BF)
    if q.numel():
        s = _steps(qkv)
        if s[2] != 1 or (s[0] | s[1]) % 8 or (B > 1 and n > 1 and s[0] != n * s[1]) or qkv.data_ptr() % 16:
            qkv = qkv[..., :3 * H * 64].clone(memory_format=torch.contiguous_format)
            s = _steps(qkv)
        ldq = s[1] if n > 1 else s[0] if B > 1 else 3 * H * 64
        _call_on(dev, "mx_rope_kv_at", qkv.data_ptr(), ldq, cs.data_ptr(), cs.shape[0], q.data_ptr(), kc.data_ptr(), vc.data_ptr(),
                 B, n, H, ctx, at.data_ptr(), at.stride(0), _int32(rot0, "rot0"))
    return q


def gemm_tile(cfg):
    import ctypes
    bm, bn = ctypes.c_int(), ctypes.c_int()
    _lib.check(_lib.load().mx_gemm_cfg_tile(cfg, ctypes.byref(bm), ctypes.byref(bn)), "mx_gemm_cfg_tile")
    return bm.value, bn.value
