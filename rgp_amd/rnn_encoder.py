"""Sequence-encoder back-constraint: the recognition model of autoreg.DeepAutoreg_rnn
(/root/reference/autoreg/rnn_encoder.py:21-150, model.py:403-440,525-551).  It stays in PyTorch-ROCm as the north star
prescribes: an fp64 stack of RNN / LSTM / GRU layers maps the raw observations (and controls) of every sequence to the
mean and softplus-variance of each hidden layer's q(X) for ALL time steps; the GP layers then run on the device through
librgp_hip.so and hand back dL/dq(X), which torch.autograd pushes into the encoder weights.

Layer l of the encoder (l = 0 is the one above the observations) takes [mean | variance] of layer l-1's output (layer 0
takes the raw [Y | U]) -- rnn_encoder.py:98-123.

The time loop of every layer (Elman/tanh RNN, LSTM or GRU cell) runs as a per-sequence persistent scan in librgp_hip.so
(rgp_rnn_scan_forward / _backward, rgp_amd/csrc/rgp_rnn.hip) when the model attached its handle: the input projections of all
time steps, the heads and every weight gradient stay (batched) torch GEMMs, only the strictly sequential recurrence moves --
the per-time-step kernel launches of the fp64 torch GRU were 95 % of a config-3 SVI step.  The parameters remain those of the
nn.RNN / nn.LSTM / nn.GRU module, so the torch path (hidden width beyond the scan's limit, no handle) and the scan are
interchangeable and are compared in tests/test_gpu_rnn.py.

rnn_type 'ssm' replaces the cell by a state-space block (MeanVarSSM) on the sequence operators of rgp_amd/seq_ops.py."""
import torch
import torch.nn as nn


def _splitk_tn(a, b, chunk=256):
    """a^T b for tall a (rows x p), b (rows x q) with a tiny p x q result: one GEMM would put the whole row sum on a single
    workgroup (0.22 ms for 4096 rows), so the sum is split into `chunk`-row pieces (batched GEMM) and added afterwards."""
    rows = a.shape[0]
    nch = rows // chunk
    body = nch * chunk
    out = a[body:].t().mm(b[body:])
    if nch > 0:
        out = out + torch.bmm(a[:body].reshape(nch, chunk, -1).transpose(1, 2), b[:body].reshape(nch, chunk, -1)).sum(0)
    return out


class _TallLinear(torch.autograd.Function):
    """y = x W^T + b for x of shape (rows, in) with many rows and few features; the weight gradient uses _splitk_tn."""

    @staticmethod
    def forward(ctx, x, W, b):
        ctx.save_for_backward(x, W)
        ctx.bias = b is not None
        return torch.addmm(b, x, W.t()) if b is not None else x.mm(W.t())

    @staticmethod
    def backward(ctx, g):
        x, W = ctx.saved_tensors
        g = g.contiguous()
        return g.mm(W), _splitk_tn(g, x), g.sum(0) if ctx.bias else None


def tall_linear(x, W, b):
    """Linear map over the last dimension of x (any leading shape)."""
    lead = x.shape[:-1]
    return _TallLinear.apply(x.reshape(-1, x.shape[-1]), W, b).view(*lead, W.shape[0])


class _RnnScanFn(torch.autograd.Function):
    """hseq = cell recurrence(gi; W_hh, b_hh) with zero initial state, gi = W_ih x + b_ih already applied; (T, B, .) layouts."""

    @staticmethod
    def forward(ctx, handle, cell, gi, W_hh, b_hh):
        from . import capi
        gi_c, W_c, b_c = gi.contiguous(), W_hh.contiguous(), b_hh.contiguous()
        hseq, gates = capi.rnn_scan_forward(handle, cell, gi_c, W_c, b_c)
        ctx.handle, ctx.cell, ctx.has_gates = handle, cell, gates is not None
        ctx.save_for_backward(W_c, b_c, hseq, *(() if gates is None else (gates,)))
        return hseq

    @staticmethod
    def backward(ctx, g_out):
        from . import capi
        saved = ctx.saved_tensors
        W_c, b_c, hseq = saved[:3]
        gates = saved[3] if ctx.has_gates else None
        dgi, dgh = capi.rnn_scan_backward(ctx.handle, ctx.cell, W_c, b_c, hseq, gates, g_out.contiguous())
        T, B, H = hseq.shape
        # dW_hh = sum_t dgh_t h_{t-1}^T (h_{-1} = 0): split-K batched GEMM, the result is only G H x H
        gW = _splitk_tn(dgh[1:].reshape(-1, dgh.shape[2]), hseq[:-1].reshape(-1, H))
        return None, None, dgi, gW, dgh.sum((0, 1))


class MeanVarRNN(nn.Module):
    """One recurrent layer with a linear mean head and a softplus variance head (rnn_encoder.py:21-83)."""

    def __init__(self, input_dim, output_dim, hidden_dim, rnn_type='rnn', bidirectional=False):
        nn.Module.__init__(self)
        cls = {'rnn': nn.RNN, 'lstm': nn.LSTM, 'gru': nn.GRU}.get(rnn_type)
        if cls is None:
            raise ValueError('Unknown rnn type')
        self.rnn = cls(input_size=input_dim, hidden_size=hidden_dim, num_layers=1, bidirectional=bidirectional)
        ndir = 2 if bidirectional else 1
        self.linear_mean = nn.Linear(hidden_dim * ndir, output_dim)
        self.linear_var = nn.Linear(hidden_dim * ndir, output_dim)
        self.soft_plus = nn.Softplus()

    handle = None               # rgp_amd.capi.Handle (set by the model): the time loops then run as device scans
    use_scan = True

    def _scan_cell(self):
        """(cell id, gate rows per unit) when this layer's recurrence fits the device scan, else None."""
        from . import _lib
        rnn = self.rnn
        if isinstance(rnn, nn.GRU):
            cell, G = _lib.CELL_GRU, 3
        elif isinstance(rnn, nn.LSTM):
            cell, G = _lib.CELL_LSTM, 4
        elif isinstance(rnn, nn.RNN) and rnn.nonlinearity == 'tanh':
            cell, G = _lib.CELL_RNN_TANH, 1
        else:
            return None
        Hh = rnn.hidden_size                       # G H lanes per step, and W_hh lives in LDS next to the step's vectors
        fits = G * Hh <= 256 and (G * Hh * (Hh | 1) + 2 * G * Hh + 2 * Hh) * 8 <= 160 * 1024
        return cell if fits else None

    def _scan(self, x, cell):
        rnn, outs = self.rnn, []
        for sfx in ([''] if not rnn.bidirectional else ['', '_reverse']):
            W_ih, W_hh = getattr(rnn, 'weight_ih_l0' + sfx), getattr(rnn, 'weight_hh_l0' + sfx)
            b_ih, b_hh = getattr(rnn, 'bias_ih_l0' + sfx), getattr(rnn, 'bias_hh_l0' + sfx)
            xs = x.flip(0) if sfx else x
            gi = tall_linear(xs, W_ih, b_ih)
            hs = _RnnScanFn.apply(self.handle, cell, gi, W_hh, b_hh)
            outs.append(hs.flip(0) if sfx else hs)
        return outs[0] if len(outs) == 1 else torch.cat(outs, dim=2)

    def forward(self, x):                       # x: (seq_len, batch, input_dim); zero initial state (h_0_type='zero')
        cell = self._scan_cell() if (self.handle is not None and self.use_scan) else None
        if cell is not None:
            out = self._scan(x, cell)
        else:
            out = self.rnn(x)[0]
        if out.is_cuda and out.shape[0] * out.shape[1] >= 1024:      # many rows, tiny heads: split-K weight gradients
            return (tall_linear(out, self.linear_mean.weight, self.linear_mean.bias),
                    self.soft_plus(tall_linear(out, self.linear_var.weight, self.linear_var.bias)))
        return self.linear_mean(out), self.soft_plus(self.linear_var(out))


class _SsmBlock(nn.Module):
    """One direction of a state-space layer, on the sequence operators of librgp_hip.so (rgp_amd/seq_ops.py):

        h = W_in x + b;   n = rms_norm(h);   [c | z] = W_uz n;   u = silu(causal convolution of c)
        [r | B | C] = W_x u;   delta = W_dt r;   y = selective scan(u, delta, A, B, C, D, z);   n' = rms_norm(W_out y + h)

    Parameters are kept in fp64 with the model's other parameters; the activations have the type of x, and the operators' parameters its
    arithmetic type."""

    N, W = 16, 4                                    # states per channel, taps of the convolution

    def __init__(self, input_dim, hidden_dim, reverse):
        nn.Module.__init__(self)
        E, N, W = hidden_dim, self.N, self.W
        R = (E + 15) // 16
        self.E, self.R, self.reverse = E, R, reverse
        self.inp = nn.Linear(input_dim, hidden_dim)
        self.norm_in = nn.Parameter(torch.ones(hidden_dim))
        self.uz = nn.Linear(hidden_dim, 2 * E, bias=False)
        self.conv_weight = nn.Parameter((torch.rand(E, W) * 2 - 1) / W ** 0.5)
        self.conv_bias = nn.Parameter((torch.rand(E) * 2 - 1) / W ** 0.5)
        self.maps = nn.Linear(E, R + 2 * N, bias=False)
        self.dt = nn.Parameter((torch.rand(E, R) * 2 - 1) / R ** 0.5)
        step = torch.exp(torch.rand(E) * 4.60517 - 6.90776)                     # softplus(dt_bias) between 1e-3 and 1e-1
        self.dt_bias = nn.Parameter(step + torch.log(-torch.expm1(-step)))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, N + 1, dtype=torch.float64)).repeat(E, 1))
        self.skip = nn.Parameter(torch.ones(E))
        self.out = nn.Linear(E, hidden_dim, bias=False)
        self.norm_out = nn.Parameter(torch.ones(hidden_dim))

    @staticmethod
    def _linear(x, W, b=None):
        W, b = W.to(x.dtype), None if b is None else b.to(x.dtype)
        rows = x.reshape(-1, x.shape[-1])                                        # one plain product, never a batched one
        tall = x.dtype == torch.float64 and rows.shape[0] >= 1024                # split-K weight gradients
        return (_TallLinear.apply(rows, W, b) if tall else nn.functional.linear(rows, W, b)).view(*x.shape[:-1], W.shape[0])

    def _parts(self, handle, x):
        from . import seq_ops
        p = (lambda t: t) if x.dtype == torch.float64 else (lambda t: t.float())
        h = self._linear(x, self.inp.weight, self.inp.bias)
        c, z = self._linear(seq_ops.rms_norm(handle, h, p(self.norm_in)), self.uz.weight).split(self.E, dim=-1)
        return p, h, c, z

    def _maps(self, u):
        r, B, Cm = self._linear(u, self.maps.weight).split((self.R, self.N, self.N), dim=-1)
        return self._linear(r, self.dt), B, Cm

    def _finish(self, handle, p, y, h):
        from . import seq_ops
        return seq_ops.rms_norm(handle, self._linear(y, self.out.weight), p(self.norm_out), residual=h)[0]

    def forward(self, handle, x, state=None, return_state=False):
        from . import seq_ops
        p, h, c, z = self._parts(handle, x)
        conv, scan = state if state is not None else (None, None)
        u = seq_ops.ssm_conv(handle, c, p(self.conv_weight), p(self.conv_bias), init=conv, reverse=self.reverse, return_state=return_state)
        u, conv = u if return_state else (u, None)
        delta, B, Cm = self._maps(u)
        y = seq_ops.ssm_scan(handle, u, delta, -torch.exp(p(self.A_log)), B, Cm, D=p(self.skip), z=z, delta_bias=p(self.dt_bias), init=scan,
                             reverse=self.reverse, return_state=return_state)
        y, scan = y if return_state else (y, None)
        n = self._finish(handle, p, y, h)
        return (n, (conv, scan)) if return_state else n

    @torch.no_grad()
    def step(self, handle, x, state):
        from . import seq_ops
        p, h, c, z = self._parts(handle, x)
        u = seq_ops.ssm_conv_step(handle, c, p(self.conv_weight), p(self.conv_bias), state[0])
        delta, B, Cm = self._maps(u)
        y = seq_ops.ssm_scan_step(handle, u, delta, -torch.exp(p(self.A_log)), B, Cm, p(self.skip), state[1], z=z, delta_bias=p(self.dt_bias))
        return self._finish(handle, p, y, h)

    def initial_state(self, batch, dtype, device):
        acc = torch.float64 if dtype == torch.float64 else torch.float32
        return (torch.zeros(batch, self.W - 1, self.E, dtype=dtype, device=device), torch.zeros(batch, self.E, self.N, dtype=acc, device=device))


class MeanVarSSM(nn.Module):
    """State-space encoder layer with the heads of MeanVarRNN.  Its recurrence is linear in the state, so it is split over time as well as
    over sequences and channels (any hidden width, any length), and it can go on from a state.  It needs the model's handle: there is no
    other path.  compute_dtype: the type of the activations inside; input, heads' output and parameters are fp64."""

    handle = None

    def __init__(self, input_dim, output_dim, hidden_dim, bidirectional=False, compute_dtype=None):
        nn.Module.__init__(self)
        self.compute_dtype = torch.float64 if compute_dtype is None else compute_dtype
        if self.compute_dtype not in (torch.float64, torch.float32, torch.bfloat16, torch.float16):
            raise ValueError('rnn_compute_dtype must be torch.float64, float32, bfloat16 or float16')
        self.blocks = nn.ModuleList([_SsmBlock(input_dim, hidden_dim, r) for r in ((False, True) if bidirectional else (False,))])
        self.linear_mean = nn.Linear(hidden_dim * len(self.blocks), output_dim)
        self.linear_var = nn.Linear(hidden_dim * len(self.blocks), output_dim)
        self.soft_plus = nn.Softplus()

    def _heads(self, n):
        n = n.double()
        lin = _SsmBlock._linear
        return lin(n, self.linear_mean.weight, self.linear_mean.bias), self.soft_plus(lin(n, self.linear_var.weight, self.linear_var.bias))

    def _need(self, online):
        if self.handle is None:
            raise RuntimeError("the 'ssm' encoder runs on librgp_hip.so: set .handle (DeepAutoreg_rnn does)")
        if online and len(self.blocks) > 1:
            raise ValueError('a bidirectional encoder reads every sequence to its end: it has no online state')

    def forward(self, x, state=None, return_state=False):                       # x: (seq_len, batch, input_dim)
        self._need(state is not None or return_state)
        x = x.to(self.compute_dtype)
        if return_state:
            n, state = self.blocks[0](self.handle, x, state, True)
            return self._heads(n) + (state,)
        ns = [b(self.handle, x, state) for b in self.blocks]
        return self._heads(ns[0] if len(ns) == 1 else torch.cat(ns, dim=2))

    def step(self, x, state):                                                   # x: (batch, input_dim); state updated in place
        self._need(True)
        return self._heads(self.blocks[0].step(self.handle, x.to(self.compute_dtype), state))

    def initial_state(self, batch):
        self._need(True)
        return self.blocks[0].initial_state(batch, self.compute_dtype, self.linear_mean.weight.device)


class SeqEncoder(nn.Module):
    """Stack of MeanVarRNN layers, lower hidden layer first (rnn_encoder.py:86-150); rnn_type 'ssm': of MeanVarSSM layers."""

    def __init__(self, input_dims, output_dims, hidden_dim, rnn_type='rnn', bidirectional=False, compute_dtype=None):
        nn.Module.__init__(self)
        assert len(input_dims) == len(output_dims)
        if compute_dtype is not None and rnn_type != 'ssm':
            raise ValueError("rnn_compute_dtype is for rnn_type 'ssm': the other cells compute in fp64")
        self.layers = nn.ModuleList()
        for l, (din, dout) in enumerate(zip(input_dims, output_dims)):
            d = din if l == 0 else 2 * din
            self.layers.append(MeanVarSSM(d, dout, hidden_dim, bidirectional, compute_dtype) if rnn_type == 'ssm' else
                               MeanVarRNN(d, dout, hidden_dim, rnn_type, bidirectional))
        self.double()

    def forward(self, x0, state=None, return_state=False):
        """(means, variances) of every layer, (seq_len, batch, H) each.  'ssm' layers: state (a list with one entry per layer, from
        ``initial_state`` or an earlier call) continues sequences; return_state=True also returns the state behind the last step."""
        online = state is not None or return_state
        if online:
            self._need_ssm()
        means, variances, states = [], [], []
        m, v = x0, None
        for l, layer in enumerate(self.layers):
            x = m if l == 0 else torch.cat((m, v), dim=2)
            if return_state:
                m, v, st = layer(x, None if state is None else state[l], True)
                states.append(st)
            else:
                m, v = layer(x, state[l]) if online else layer(x)
            means.append(m)
            variances.append(v)
        return (means, variances, states) if return_state else (means, variances)

    def _need_ssm(self):
        if not all(isinstance(layer, MeanVarSSM) for layer in self.layers):
            raise ValueError("only rnn_type 'ssm' encoders go on from a state")

    def initial_state(self, batch):
        """The state before the first observation of ``batch`` sequences."""
        self._need_ssm()
        return [layer.initial_state(batch) for layer in self.layers]

    @torch.no_grad()
    def step(self, x, state):
        """One observation of every sequence: x (batch, input_dim) -> (means, variances) of every layer, (batch, H) each; state is updated
        in place."""
        self._need_ssm()
        means, variances = [], []
        m, v = x, None
        for l, layer in enumerate(self.layers):
            m, v = layer.step(m if l == 0 else torch.cat((m, v), dim=1), state[l])
            means.append(m)
            variances.append(v)
        return means, variances
