// HipScoring.cs -- the scoring operators of HipExecutionProvider, which have no counterpart among the reference's:
// 8-bit floating point codes with a Float scale for each block of 128 (QuantizeBlocks), their product
// (MatMulBlocks), and what logits say about tokens (TokenLogProbs).  The library checks every argument; its messages
// become the OpResult's.  Profiles chart them under the operator they stand beside: Cast, MatMul and Softmax.
// Belongs in src/Lokad.Onnx.Backend.
namespace Lokad.Onnx;

using System;
using System.Linq;

using static OpResult;

public unsafe partial class HipExecutionProvider
{
    /// <summary>Element type codes of the 8-bit floating types (ONNX TensorProto.DataType): tensors of them exist
    /// on the device only, as QuantizeBlocks' outputs and MatMulBlocks' operands.</summary>
    public const long Float8E4M3FN = 17, Float8E5M2 = 19;

    static OpResult Scored(OpType op, int st, params LxTensor[] outputs)
    {
        if (st == 0)
            return new OpResult { Op = op, Status = OpStatus.Success, Outputs = outputs.Select(y => (ITensor)DeviceTensor.Own(y)).ToArray() };
        return Failure(op, HipNative.LastError());
    }

    /// <summary>Codes and scales of X: a scale for each 1x128 (blockRows 1) or 128x128 (blockRows 128) block of its
    /// last axes.</summary>
    public static OpResult QuantizeBlocks(ITensor? X, long to = Float8E4M3FN, long blockRows = 1)
    {
        var op = OpType.Cast;
        if (X is null) return MissingInput(op, nameof(X));
        using var args = new Args();
        LxTensor x = args.In(X), q = default, s = default;
        MathStage();
        var st = HipNative.lx_QuantizeBlocks(&x, to, blockRows, &q, &s);
        return Scored(op, st, q, s);
    }

    /// <summary>A [..., M, K] times B [N, K] by output channel, both of 8-bit codes with their blocks' scales, plus a
    /// bias row.</summary>
    public static OpResult MatMulBlocks(ITensor? A, ITensor? aScale, ITensor? B, ITensor? bScale, ITensor? bias = null)
    {
        var op = OpType.MatMul;
        if (A is null) return MissingInput(op, nameof(A));
        if (aScale is null) return MissingInput(op, nameof(aScale));
        if (B is null) return MissingInput(op, nameof(B));
        if (bScale is null) return MissingInput(op, nameof(bScale));
        using var args = new Args();
        LxTensor a = args.In(A), sa = args.In(aScale), b = args.In(B), sb = args.In(bScale), y = default;
        LxTensor c = bias is null ? default : args.In(bias);
        MathStage();
        var st = HipNative.lx_MatMulBlocks(&a, &sa, &b, &sb, bias is null ? null : &c, &y);
        return Scored(op, st, y);
    }

    /// <summary>Of each row of logits: the log-probability of its id (with ids), the entropy (with entropy), the most
    /// probable ids and their log-probabilities (with top); the outputs asked for, in that order.</summary>
    public static OpResult TokenLogProbs(ITensor? logits, ITensor? ids = null, long top = 0, bool entropy = false)
    {
        var op = OpType.Softmax;
        if (logits is null) return MissingInput(op, nameof(logits));
        using var args = new Args();
        LxTensor x = args.In(logits), lp = default, h = default, ti = default, tl = default;
        LxTensor i = ids is null ? default : args.In(ids);
        MathStage();
        var st = HipNative.lx_TokenLogProbs(&x, ids is null ? null : &i, top, ids is null ? null : &lp,
                                            entropy ? &h : null, top == 0 ? null : &ti, top == 0 ? null : &tl);
        var asked = new (bool, LxTensor)[] { (ids is not null, lp), (entropy, h), (top != 0, ti), (top != 0, tl) };
        return Scored(op, st, asked.Where(o => o.Item1).Select(o => o.Item2).ToArray());
    }
}
