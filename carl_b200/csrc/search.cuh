// Launch wrappers of the search operators (search.cu): beam selection and state
// reordering.
#pragma once

#include <cstdint>

#include <cuda_runtime.h>

namespace cb {

constexpr int BEAM_MAX_BEAMS = 1024;   // beams of a group
constexpr int BEAM_MAX_WIDTH = 128;    // continuations kept per group
constexpr int JOINT_MAX_BEAMS = 32;    // the same over the action heads
constexpr int JOINT_MAX_WIDTH = 32;

enum LogitType : int { LOGITS_F32 = 0, LOGITS_BF16 = 1, LOGITS_F16 = 2 };

struct BeamParams
{
    const void* logits;                 // [groups, beams, vocab], last dimension dense
    long long groupStride, beamStride;  // elements
    const float* scores;                // [groups, beams]
    const uint8_t* mask;                // [groups, beams, vocab] or null; 0 = not allowed
    long long maskGroupStride, maskBeamStride;
    const uint8_t* finished;            // [groups, beams] or null
    float* outScores;                   // [groups, width]
    long long* outParents;
    int* outActions;                    // [groups, width] (joint: [groups, width, 7])
    double* sum;                        // workspace: [rows, segs] sum of exp(logit - top)
    float* top;                         // [rows, segs] largest logit
    float* chunks;                      // [rows, segs, 32] largest logit of each lane's part
    int groups, beams, vocab, width;
    int segVectors;                     // 16-byte vectors of a segment
    int segs;                           // warps to a row; 0: a block to a group
};

// Workspace bytes of a flat selection, and its pointers into `base`; sets p.segs.
long long planBeamSelect(BeamParams& p, LogitType type, void* base);
void launchBeamSelect(const BeamParams& p, LogitType type, cudaStream_t s);
void launchJointSelect(const BeamParams& p, LogitType type, cudaStream_t s);

// One state array: `outer` slabs of groups * beams rows of `inner` bytes.
struct StateArray
{
    void* data;
    long long outer, outerStride, inner;  // slabs, bytes between slabs, bytes per row
};

// new[o, g, j] = old[o, g, parents[g, j]], in place.
void launchReorder(const StateArray* arrays, int count, const long long* parents, int groups, int beams, cudaStream_t s);

// After the reordering of an env's words: the env-global car index of each moved
// car's last bump victim (one word per car) points into the car's new sim.
void launchMoveContacts(int* contact, const long long* parents, int nSim, int beams, int nCars, cudaStream_t s);

}  // namespace cb
