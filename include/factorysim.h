/* factorysim.h -- C ABI of the MI355X-native batched factory-manipulation environment.
 *
 * Drop-in boundary for the reference's env-step path.  The reference exposes it as a Gymnasium env
 * stepped through stable-baselines3's VecEnv (SubprocVecEnv, one Python process per arena):
 *   FactoryManipulationEnv.step(action)         /root/reference/src/environments.py:151-202
 *   FactoryManipulationEnv.reset(seed, options) /root/reference/src/environments.py:204-248
 *   BaseEnv.step_sim / reset_sim                 /root/reference/challenge_env/challenge_env/base_env.py:177-282
 *   make_vec_env(..., vec_env_cls=SubprocVecEnv) /root/reference/src/learning.py:98-100
 * This ABI replaces the whole SubprocVecEnv fan-out: one handle owns N arenas resident in HBM and
 * one fm_step() advances all of them by one env-step (100 physics substeps + task layer + wrappers,
 * with SB3-style auto-reset).  factory_marl_amd/vec_env.py binds it with ctypes; INTEGRATION.md
 * shows the binding a maintainer of the reference would add.
 *
 * Conventions
 *  - Status codes: 0 = ok, < 0 = error (FM_E*); fm_last_error() returns a thread-local message.
 *    No C++ exception crosses the ABI.
 *  - Ownership: the library owns all arena state (device memory).  The caller owns every I/O
 *    buffer passed in and keeps it alive for the call; I/O buffers are DEVICE pointers
 *    (e.g. torch.Tensor.data_ptr() of a ROCm tensor) unless a parameter says "host".
 *  - Streams: each handle runs on one HIP stream (fm_set_stream); calls are asynchronous on it.
 *    A handle is not re-entrant; several handles (one per GPU / rank) may be driven concurrently.
 *  - Errors are reported eagerly for argument problems; device faults surface on fm_sync().
 */
#ifndef FACTORYSIM_H
#define FACTORYSIM_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define FM_OK 0
#define FM_EINVAL (-1)  /* bad argument / config */
#define FM_EDEVICE (-2) /* HIP runtime error */
#define FM_ENOMEM (-3)
#define FM_ESTATE (-4)  /* call order (e.g. step before reset) */

/* env classes of src/environments.py whose step() this library implements.  Actions are float32 [N, act_dim]:
 *   FACTORY                  act_dim 0  (every arm on the IK base policy; pass any pointer, it is not read)
 *   SINGLEFULLRL, SINGLEDELTA act_dim 8  (Box[-1, 1])
 *   ALLFULLRL, ALLDELTA       act_dim 8A (Box[-1, 1])
 *   PAUSE / BACKUP_IK_TOGGLE  act_dim A  (MultiDiscrete([2] * A) as 0.0 / 1.0; 1.0 = follow the IK proposal)
 * Observations are 24A + 13K float32 (+ 8A IK proposals for the two toggle classes). */
#define FM_ENV_FACTORY 0              /* FactoryManipulationEnv: IK on every arm, score-delta reward (environments.py:25-248) */
#define FM_ENV_ALLFULLRL_PROGRESS 1   /* AllFullRLProgressRewardEnv (environments.py:462-495) */
#define FM_ENV_SINGLEFULLRL_PROGRESS 2 /* SingleFullRLProgressRewardEnv (environments.py:386-420) */
#define FM_ENV_SINGLEDELTA_PROGRESS 3 /* SingleDeltaProgressRewardEnv (environments.py:423-459) */
#define FM_ENV_ALLDELTA_PROGRESS 4    /* AllDeltaProgressRewardEnv (environments.py:498-535) */
#define FM_ENV_PAUSE_IK_TOGGLE 5      /* PauseIKToggleEnv (environments.py:538-612) */
#define FM_ENV_BACKUP_IK_TOGGLE 6     /* BackupIKToggleEnv (environments.py:615-645) */

#define FM_FP32 0 /* physics state and arithmetic in float  (north-star configuration) */
#define FM_FP64 1 /* physics state and arithmetic in double (bit-for-bit twin of the oracle's precision) */

/* Mirrors BaseEnv.__init__ kwargs (base_env.py:15-35) and ProgressRewardEnv weights
 * (environments.py:252-258).  fm_config_default() fills the reference defaults. */
typedef struct fm_config {
  int32_t num_arenas;
  int32_t num_arms;        /* even, >= 2 (scene.py:149) */
  int32_t max_num_objects; /* K cubes per arena */
  int32_t env_class;       /* FM_ENV_* */
  int32_t precision;       /* FM_FP32 / FM_FP64 */
  int32_t max_contacts;    /* per-arena contact capacity (0 = automatic) */
  double initial_conveyor_speed;  /* 0.1 m/s */
  double conveyor_acceleration;   /* 0.001 m/s^2 */
  double pt_time;                 /* 0.2 s */
  double force_contact_threshold; /* 200 N */
  double control_frequency;       /* 10 Hz -> frame_skip = int((1/f)/0.001) = 100 */
  double spawn_freq;              /* 0.1 (multiplied by num_arms, base_env.py:36) */
  double spawn_freq_increase;     /* 1.001 */
  double gripper_to_closest_cube_reward_factor;
  double closest_cube_to_bucket_reward_factor;
  double small_action_norm_reward_factor;
  double base_reward;
  int32_t solver_iterations; /* Newton iterations cap (MuJoCo default 100) */
  double solver_tolerance;   /* scaled improvement / gradient tolerance (MuJoCo default 1e-8) */
  int32_t obs_float64;       /* 1: obs / terminal_obs rows are float64 (the toggle classes' observation dtype in the
                                reference: float32 state columns widened, float64 IK proposals, environments.py:576);
                                0: float32 rows (default) */
} fm_config;

/* Per-step info, all DEVICE pointers, any may be NULL (info dict of base_env.py:274-280 plus the
 * SB3 Monitor / auto-reset extras). */
typedef struct fm_info {
  int32_t* scores;          /* [N, 2] */
  int32_t* num_obj;         /* [N]   objects in scene after the step */
  double* play_time;        /* [N] */
  double* conveyor_speed;   /* [N] */
  uint8_t* out_of_reach;    /* [N]   TaskManager.terminate */
  uint8_t* force_terminate; /* [N] */
  void* terminal_obs;       /* [N, obs_dim] float32 (float64 with obs_float64) written for arenas that terminated
                             (before auto-reset) */
  double* episode_return;   /* [N]   Monitor "r" of the finished episode (valid where terminated) */
  int32_t* episode_length;  /* [N]   Monitor "l" */
  int32_t* terminal_scores; /* [N, 2] scores of the finished episode (ep_score_history entry) */
} fm_info;

typedef struct fm_handle fm_handle;

/* ABI version of this header and the size of the fm_config the library was built with: a binding built against a
 * different header checks both before fm_create (version 2 appended fm_config.obs_float64; a caller passing the
 * version-1 struct would leave it unset).  factory_marl_amd/_lib.py refuses a library whose version or fm_config size
 * differs from its own. */
#define FM_ABI_VERSION 2
int fm_abi_version(void);
int fm_config_size(void);

void fm_config_default(fm_config* cfg);

/* Create N arenas on `device`.  seeds: host array [N] -- per-arena seed used, as in the reference,
 * both for build_scene's cube sizes (scene.py:121) and for the TaskManager RNG (task_utils.py:19).
 * NULL = every arena uses seed 42 (the value in every saved run config under runs/).
 * device = -1: the CPU backend -- the same kernels on host threads, every buffer argument of the
 * handle's calls host memory, results identical in meaning (reference config 1: visualisation.py:32-77 steps one env
 * on the CPU); fm_render and fm_profile return FM_EINVAL.  A GPU device that is absent is FM_EDEVICE, never a CPU
 * fallback. */
int fm_create(const fm_config* cfg, int device, const uint64_t* seeds, fm_handle** out);
void fm_destroy(fm_handle* h);
const char* fm_last_error(void);

/* Set the HIP stream all later calls of this handle run on (hipStream_t passed as void*; NULL = the
 * legacy default stream).  fm_create starts on a private non-blocking stream. */
int fm_set_stream(fm_handle* h, void* stream);
int fm_sync(fm_handle* h);

/* Runtime-mutable scalars (SB3 VecEnv.set_attr / get_attr on the reference env's attributes, base_env.py:133-141,
 * environments.py:276-282): "pt_time", "initial_conveyor_speed", "conveyor_acceleration",
 * "force_contact_threshold", "spawn_freq_increase", "init_spawn_freq" (= spawn_freq * num_arms),
 * "gripper_to_closest_cube_reward_factor", "closest_cube_to_bucket_reward_factor",
 * "small_action_norm_reward_factor", "base_reward".  Global to the handle; launches queued after the call use the
 * new value.  control_frequency (frame_skip), num_arms, max_num_objects and seeds are fixed at fm_create.
 * Per-arena dynamic values (play_time, conveyor_speed, spawn_freq) live in the state record (fm_set_state).
 * "experiment_flags": the kernel's experiment switches (A/B probes and equivalence tests only; 0 in production),
 * initialised once at fm_create from FM_* environment variables. */
int fm_set_param(fm_handle* h, const char* name, double value);
int fm_get_param(const fm_handle* h, const char* name, double* value);

int fm_obs_dim(const fm_handle* h);
int fm_act_dim(const fm_handle* h);
int fm_num_arenas(const fm_handle* h);
int fm_nq(const fm_handle* h);
int fm_nv(const fm_handle* h);
int fm_nu(const fm_handle* h);
int fm_workspace_bytes(const fm_handle* h); /* LDS bytes of one arena's env-step workspace */

/* reset(): reset arenas where mask[i] != 0 (device uint8 [N]; NULL = all) and write their obs.
 * Mirrors BaseEnv.reset_sim + FactoryManipulationEnv.reset (environments.py:204-248): the
 * TaskManager RNG is NOT reseeded (task_utils.py:19), progress-reward distance memories persist. */
int fm_reset(fm_handle* h, const uint8_t* mask, void* obs);

/* step(): actions float32 [N, act_dim] (device).  Writes obs [N, obs_dim] (float32, or float64 with
 * cfg.obs_float64; reset obs for arenas that terminated), reward [N], terminated [N], truncated [N] (always 0: the
 * reference has no time limit, environments.py:202), and info.  Any output pointer may be NULL. */
int fm_step(fm_handle* h, const float* actions, void* obs, float* reward, uint8_t* terminated,
            uint8_t* truncated, const fm_info* info);

/* Teacher forcing / checkpointing of the full arena state (HOST buffers).
 * Physics block per arena (float64): qpos[nq], qvel[nv], qpos_stage[nq], qvel_stage[nv],
 * qacc_warmstart[nv], ctrl_target[nu]; see fm_state_layout() for the task block. */
int fm_state_size(const fm_handle* h);                 /* bytes per arena of the exported record */
int fm_get_state(fm_handle* h, void* host_out);        /* [N * fm_state_size] */
int fm_set_state(fm_handle* h, const void* host_in);

/* Diagnostics: per-arena counters accumulated since create (host [N * fm_num_counters()] int64):
 * [0] contacts dropped for capacity, [1] Newton iterations, [2] solver max-iteration hits,
 * [3] bucket-index anomalies (task_utils.py:103-113 would raise IndexError),
 * [4] contacts summed over physics stages, [5] most contacts in one stage (both before any capacity
 * cut), [6] objects in scene summed over env-steps, [7] episodes ended (terminations),
 * [8] env-steps rerun by the (2,4) scene's wide-capacity kernel (a stage above 64 contacts; the Newton counters
 * [1] [2] then include the abandoned part of the step). */
int fm_get_counters(fm_handle* h, int64_t* host_out);
int fm_num_counters(void);
/* Diagnostic: each arena's last env-step duration in GPU wall-clock ticks (host [N] uint32; 0 until its first step;
 * the longest-first dispatch order of the next step is sorted by these) -- the launch's load balance. */
int fm_get_costs(fm_handle* h, uint32_t* host_out);
/* Measurement: time each env-step kernel launch alone with a HIP event pair on the handle's stream (enable != 0;
 * enabling or disabling discards earlier records).  fm_get_kernel_time synchronises the stream and returns the
 * summed duration of the step-kernel launches recorded since the last read (the longest-first order kernel, the
 * rerun-list reset and the (2,4) wide rerun launch are outside the pairs), then starts a new record.  bench.py's
 * roofline.achieved divides the algorithmic bytes by this per-launch time. */
int fm_kernel_timing(fm_handle* h, int enable);
int fm_get_kernel_time(fm_handle* h, double* total_ms, int* launches);

/* Diagnostic: wall-clock phase profile of fm_step summed over arenas (host [24] uint64).
 * mode 1 = zero and enable, 0 = disable, -1 = leave as is; host_out (may be NULL) receives the
 * totals: [0..13] clock ticks per phase (FK, geoms+M, collision's contact ranking, constraint rows, smooth acc,
 * Newton setup / gradient / Hessian / Cholesky / solve / line search / final forces, integration,
 * task+obs), [14] sum of ncon over stages, [15] the clock rate in kHz, [16..18] the rest of the collision phase:
 * geom centres + body bounds, body-pair midphase, geom-pair expansion + narrowphase; [19..22] the dense blocked
 * Cholesky's diagonal blocks, panels, trailing updates and substitutions (scenes above 80 dofs, else 0); [23] zero. */
int fm_profile(fm_handle* h, int mode, uint64_t* host_out);

/* Diagnostic (tests only): recompute one mj_step1 + acceleration stage of `arena` at its stored stage
 * state and dump internals as float64 into host_out (capacity `cap` doubles).  Returns the number of
 * doubles written (< 0 on error).  Layout in factory_marl_amd/csrc/fm_device.hpp (debug_kernel). */
int fm_debug_dump(fm_handle* h, int arena, int actuated, double* host_out, int cap);

/* Offscreen rgb_array rendering (rendering.py:153-305 OffScreenViewer, 653-789 MujocoRenderer.render;
 * base_env.py:288-306 render()), batched: `count` arenas (host int32 indices) at their current state are ray
 * cast on the GPU into the device buffer rgb [count][height][width][3] uint8, row 0 = top (rgb_array layout).
 * camera: host float[6] = lookat xyz, distance, azimuth, elevation (degrees; MuJoCo free-camera convention), or
 * NULL for the reference viewer's initial camera (scene.py:164-169); fovy 45.  Drawn is the collision geometry
 * the physics uses (arms as their collision spheres and gripper boxes).  geom_frames (optional device buffer,
 * float [count][fm_render_ngeom][20]: MuJoCo geom id, type 0 plane / 1 sphere / 2 box, world pos[3], R[9]
 * row-major, half sizes[3], rgb[3]) receives the geometry the image was cast from; rgb may be NULL to get only
 * those.  Asynchronous on the handle's stream (the arena list is copied before the call returns). */
int fm_render(fm_handle* h, const int32_t* arenas, int count, int width, int height, const float* camera,
              uint8_t* rgb, float* geom_frames);
int fm_render_ngeom(const fm_handle* h); /* collidable geoms per arena (rows of geom_frames) */

/* Scene export (host only, no device needed): the scene fm_create builds for (num_arms,
 * max_num_objects) with the cubes of arena seed `seed`, as one flat MJCF document -- the model
 * build_scene(num_objects, seed=seed, num_arms) (challenge_env/scene.py:109-161) compiles to under
 * dm_control, with its element names (base_env.py:114-126, ik_policy.py:41-45) and id order, for an
 * optional MuJoCo cross-check.  meshdir: directory of the iiwa14 .obj files (visual meshes), or
 * NULL/"" for non-colliding placeholders in the same geom slots.  *len receives the document length;
 * with buf == NULL only the length is returned; otherwise cap must be >= *len + 1 (NUL-terminated). */
int fm_scene_mjcf(int num_arms, int max_num_objects, uint64_t seed, const char* meshdir, char* buf, size_t cap,
                  size_t* len);

/* ---------------------------------------------------------------------------------------------------------------
 * Policy-head operators: layer norm, drawing categories from logits, distillation from a teacher's top logits.
 * They need no handle.  Conventions:
 *  - `device` is a GPU ordinal (buffers are device pointers, the work is queued on `stream`, a hipStream_t of that
 *    device or NULL for its default stream; the caller's current device is left as it was) or -1, the CPU backend (host pointers, done on
 *    return).
 *  - Rows: `*_stride` is the distance of consecutive rows in elements (>= 0; 0 = every row the same), elements of one
 *    row are adjacent.  Outputs are contiguous.  No alignment beyond the element's own is needed.
 *  - Nothing is allocated, synchronised or kept between calls, so every call can be captured into a graph; the
 *    workspace (fm_*_workspace bytes, 16-byte aligned, contents ignored) belongs to one call at a time.
 *  - rows = 0 is valid and does nothing but zero a sum over rows.  Arguments are checked before anything runs:
 *    FM_EINVAL, no output touched. */
#define FM_MAX_COLS (1 << 28) /* the most elements of a row: kernels count them, twice over and a block more, in 32 bits */
#define FM_DTYPE_F32 0
#define FM_DTYPE_F16 1
#define FM_DTYPE_BF16 2
#define FM_DTYPE_F64 3 /* uniform numbers */
#define FM_DTYPE_I32 4 /* category indices */
#define FM_DTYPE_I64 5

/* y = (x - mean) * rstd * weight + bias over the last dimension, rstd = 1 / sqrt(variance + eps), biased variance;
 * statistics and sums in 32 bits.  x, y, dy, dx are of x_dtype; weight, bias and their gradients of param_dtype
 * (x_dtype or F32). */
typedef struct fm_layer_norm_args {
  int32_t device, x_dtype, param_dtype, reserved;
  int64_t rows, cols; /* 1 <= cols <= FM_MAX_COLS */
  const void* x;
  int64_t x_stride;
  const void* weight; /* [cols]; NULL = ones */
  const void* bias;   /* [cols]; NULL = zeros (forward only) */
  double eps;         /* >= 0 (forward only) */
  void* y;            /* forward: [rows, cols] */
  float* mean;        /* [rows]: written by the forward call (both NULL: not kept), read by the backward call */
  float* rstd;
  const void* dy; /* the rest: backward only */
  int64_t dy_stride;
  void* dx;      /* [rows, cols]; NULL = not wanted */
  void* dweight; /* [cols]; NULL = not wanted */
  void* dbias;   /* [cols]; NULL = not wanted */
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} fm_layer_norm_args;
int fm_layer_norm_forward(const fm_layer_norm_args* a);
/* dx, dweight, dbias from dy; the sums over rows are taken in a fixed order (the same inputs give the same bits) */
int fm_layer_norm_backward(const fm_layer_norm_args* a);
int64_t fm_layer_norm_workspace(int64_t rows, int64_t cols);

/* Draws one category of each row: the row's categories are ranked by logit, the lower index first among equals, and
 * weigh w = exp((logit - largest) / temperature).  Kept are the first top_k, of those the shortest leading part that
 * holds at least top_p of their weight (the product as a double), of those the ones with w >= min_p; out is the first of
 * the kept ones up to which more than u of their weight lies.  mask (bytes, 0 = barred; any value may stand in a barred logit) and logits
 * of -inf bar a category; +inf outweighs everything finite.  A row with nothing left, with NaN in a logit that is not
 * barred or with a NaN setting gives -1.  Each setting is one number for all rows, or, where *_rows is not NULL, a float
 * (top_k: int32) of each row's own.
 * temperature <= 0: the largest logit; top_k <= 0, top_p >= 1, min_p <= 0: off; top_p <= 0 and min_p >= 1 keep the
 * largest (min_p: and its equals); u is meant to be in [0, 1) and is cut to what is kept.  Weights are whole multiples of
 * 2^-s of the largest's, s = 51 or what 62 bits leave for the sum of cols of them (45 for 2^17 categories), and are added up as
 * whole numbers, so a call gives the same on every run.  What weighs less than 2^-(s+1) is never drawn, on the GPU beyond
 * 2048 columns nor what weighs less than e^-33.  Weights are good to 6e-15 of themselves, the GPU's sums beyond 2048
 * columns to 5e-13: the GPU and the CPU can draw neighbours where a border lies as near as that to one between two
 * categories (shares of equal logits that hold all the weight are exact). */
typedef struct fm_sample_args {
  int32_t device, dtype, u_dtype, reserved; /* u_dtype: F32 or F64 */
  int64_t rows, cols;                       /* 1 <= cols <= FM_MAX_COLS */
  const void* logits;
  int64_t stride;
  const uint8_t* mask; /* [rows, cols] with mask_stride; NULL = none */
  int64_t mask_stride;
  const void* u; /* [rows] */
  double temperature, top_p, min_p;
  int64_t top_k;
  const float* temperature_rows;
  const float* top_p_rows;
  const float* min_p_rows;
  const int32_t* top_k_rows;
  int64_t* out; /* [rows] */
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} fm_sample_args;
int fm_sample_logits(const fm_sample_args* a);
int64_t fm_sample_workspace(int64_t rows, int64_t cols); /* 0: a draw takes none, workspace is not read */

/* loss[i] = T^2 * sum over the listed entries of p (log p - log q[index]), q = softmax(logits / T) over all columns,
 * p = softmax(teacher / T) over the row's listed entries.  An entry with a negative index or a teacher logit of -inf
 * is not listed; a row without entries has loss 0 and gradient 0; an index >= cols makes the row's loss and
 * gradient NaN, and so does a row without a softmax (logits all -inf, or +inf or NaN among them; +inf or NaN among the listed
 * teacher logits); the same index listed twice counts twice.  Backward: dlogits = grad[i] * T * (q - p at the listed places). */
typedef struct fm_distill_args {
  int32_t device, dtype, index_dtype, teacher_dtype; /* index_dtype: I32 or I64; teacher: F32, F16 or BF16 */
  int64_t rows, cols, k;                             /* 1 <= cols <= FM_MAX_COLS, 1 <= k <= FM_DISTILL_MAX_K */
  const void* logits;
  int64_t stride;
  const void* index; /* [rows, k] */
  int64_t index_stride;
  const void* teacher; /* [rows, k] */
  int64_t teacher_stride;
  double temperature; /* > 0 */
  float* loss;        /* forward: [rows] */
  float* stats;       /* [rows, 2], largest logit and sum of exp: written by the forward call (NULL: not kept), read
                         * by the backward call */
  const float* grad;  /* backward: [rows] with grad_stride */
  int64_t grad_stride;
  void* dlogits; /* backward: [rows, cols] */
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} fm_distill_args;
#define FM_DISTILL_MAX_K 1024
int fm_distill_forward(const fm_distill_args* a);
int fm_distill_backward(const fm_distill_args* a);
int64_t fm_distill_workspace(int64_t rows, int64_t cols);

#ifdef __cplusplus
}
#endif
#endif
